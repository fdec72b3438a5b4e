"""The measured cases of the operators of a post-training step: per-head query / key RMSNorm with the rotary position
rotation (one to four position axes), the rotation alone, the clipped policy loss and the preference loss on logits.

``run`` computes a case in plain torch operations when ``own`` is false, and through the framework's entry points when
it is true. ``exact`` is the same result from the definition in 64 bits (rotation as a complex product, gradients by
differentiation)."""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
IGNORED = -100
EPS = 1e-6
CLIP_LOW, CLIP_HIGH, KL_COEF, TEMPERATURE = 0.2, 0.28, 0.05, 0.9
BETA, SMOOTHING = 0.1, 0.05
LARGEST_LOGITS = 8192 * 128256


# ---------------------------------------------------------------- cases

def _heads(name, op, way, dtype, batch, seq, hq, hk, dim, rot, axes=1, interleaved=False, fused=True, far=0):
    """A case of qk_norm_rope or rope: [batch, seq] tokens of hq query and hk key heads of `dim` features, `rot` of
    them rotated; `fused`: q and k are views into one projection output; positions start at `far`."""
    return {"name": name, "op": op, "way": way, "dtype": dtype, "batch": batch, "seq": seq, "hq": hq, "hk": hk,
            "dim": dim, "rot": rot, "axes": axes, "interleaved": interleaved, "fused": fused, "far": far}


def _loss(name, op, way, dtype, rows, cols, ignored, pad=0, pairs=0, tail=0):
    """A case of policy_loss or preference_loss: logits [rows, cols] in a matrix of cols + pad columns, `ignored` rows
    left out; preferences: `pairs` pairs of sequences over rows - tail rows."""
    return {"name": name, "op": op, "way": way, "dtype": dtype, "rows": rows, "cols": cols, "ignored": ignored,
            "pad": pad, "pairs": pairs, "tail": tail}


def listed():
    return [
        # one decoded token of one sequence, deep in a long context: latency
        _heads("qk_norm_rope_token", "qk_norm_rope", "fwd", "bf16", 1, 1, 32, 8, 128, 128, far=131071),
        # a long prompt, q and k as the projection wrote them
        _heads("qk_norm_rope_prompt", "qk_norm_rope", "fwd", "bf16", 1, 16384, 32, 8, 128, 128),
        # a ragged batch of a small model that rotates half of each head, neighbours paired
        _heads("qk_norm_rope_partial", "qk_norm_rope", "fwd", "fp16", 3, 1111, 12, 3, 80, 40, interleaved=True),
        # the backward pass of a training batch
        _heads("qk_norm_rope_train", "qk_norm_rope", "bwd", "bf16", 4, 4096, 32, 8, 128, 128),
        # the backward pass of a small 32-bit run
        _heads("qk_norm_rope_train_fp32", "qk_norm_rope", "bwd", "fp32", 2, 777, 8, 8, 64, 64, fused=False),
        # a video: time, height and width of each patch
        _heads("rope_video", "rope", "fwd", "bf16", 1, 29971, 16, 16, 128, 128, axes=3),
        # the backward pass of image patches, height and width, a head size with an odd number of 16-byte vectors
        _heads("rope_image_train", "rope", "bwd", "fp16", 5, 1369, 16, 16, 72, 72, axes=2, fused=False),
        # a few rows of a small policy in 32 bits: latency
        _loss("policy_small", "policy_loss", "fwd_bwd", "fp32", 8, 1000, 1),
        # one micro-batch's update of a policy, prompt rows left out
        _loss("policy_update", "policy_loss", "fwd_bwd", "bf16", 8192, 128256, 1024),
        # the losses of an evaluation, a vocabulary of odd length, rows padded to a multiple of 64
        _loss("policy_eval_odd", "policy_loss", "fwd", "fp16", 1023, 32001, 200, pad=63),
        # the forward pass over sixteen pairs
        _loss("preference_batch", "preference_loss", "fwd", "bf16", 6000, 128256, 1500, pairs=16),
        # its backward pass over four pairs, a padded batch whose last rows belong to no sequence
        _loss("preference_train", "preference_loss", "bwd", "bf16", 2100, 128256, 500, pairs=4, tail=52),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    op = rng.choice(["qk_norm_rope", "qk_norm_rope", "rope", "policy_loss", "policy_loss", "preference_loss"])
    if op in ("qk_norm_rope", "rope"):
        dim = rng.choice([64, 72, 80, 96, 128, 128, 192, 256])
        axes = rng.choice([1, 1, 2, 3, 4] if op == "qk_norm_rope" else [1, 2, 3, 4])
        rot = dim if rng.random() < 0.7 else dim // 2
        hk = rng.choice([1, 2, 3, 4, 8, 16])
        hq = hk * rng.choice([1, 2, 4, 5])
        most = 16384 * 40 * 128 // ((hq + hk) * dim * (2 if dtype == "fp32" else 1))
        batch = rng.choice([1, 1, 2, 3, 7])
        seq = max(1, _log_uniform(rng, 1, most) // batch)
        case = _heads("", op, rng.choice(["fwd", "bwd"]), dtype, batch, seq, hq, hk, dim, rot, axes, rng.random() < 0.3,
                      rng.random() < 0.6, rng.choice([0, 0, 4000, 1000003]))
    else:
        cols = _log_uniform(rng, 500, 128256)
        most = LARGEST_LOGITS // (cols * (2 if dtype == "fp32" else 1) * 2)
        pairs = 0 if op == "policy_loss" else rng.choice([1, 2, 5, 16, 33])
        rows = max(2 * pairs, _log_uniform(rng, 1, min(most, 40000)))
        ignored = int(rows * rng.choice([0.0, 0.05, 0.3]))
        tail = int(rows * 0.03) if pairs and rng.random() < 0.5 else 0
        ways = ["fwd", "bwd", "fwd_bwd"] if op == "policy_loss" else ["fwd", "bwd"]
        case = _loss("", op, rng.choice(ways), dtype, rows, cols, min(ignored, rows - tail), rng.choice([0, 0, -cols % 64]),
                     pairs, tail)
    del case["name"]
    return case


# ---------------------------------------------------------------- inputs

def _sections(case):
    """Frequencies of each axis: the first axis has what the others leave."""
    half, axes = case["rot"] // 2, case["axes"]
    if axes == 1:
        return None
    each = (half * 3) // (4 * axes - 1) if axes > 2 else half // 2
    return (half - each * (axes - 1),) + (each,) * (axes - 1)


def _positions(case, g):
    """[batch, seq] positions, or [axes, batch, seq]: the first axis counts on, the others walk over a grid."""
    b, s = case["batch"], case["seq"]
    t = torch.arange(s, device="cuda") + case["far"]
    if case["axes"] == 1:
        return (t + torch.randint(0, 17, (b, 1), generator=g, device="cuda")).contiguous()
    side = 37
    walk = [t // (side * side), (t // side) % side, t % side, t % 5][:case["axes"]]
    return torch.stack(walk).unsqueeze(1).expand(-1, b, -1).contiguous()


def _prepare_heads(case, g):
    dt, b, s, d = DTYPES[case["dtype"]], case["batch"], case["seq"], case["dim"]
    hq, hk = case["hq"], case["hk"]
    rand = lambda *shape: torch.randn(*shape, generator=g, device="cuda")  # noqa: E731
    st = {"case": case, "positions": _positions(case, g), "sections": _sections(case)}
    if case["fused"]:
        qkv = rand(b, s, (hq + 2 * hk) * d).to(dt)
        st["q"] = qkv[..., :hq * d].unflatten(-1, (hq, d))
        st["k"] = qkv[..., hq * d:(hq + hk) * d].unflatten(-1, (hk, d))
    else:
        st["q"], st["k"] = rand(b, s, hq, d).to(dt), rand(b, s, hk, d).to(dt)
    st["q_weight"], st["k_weight"] = (1 + 0.1 * rand(d)).to(dt), (1 + 0.1 * rand(d)).to(dt)
    n = case["rot"] // 2
    st["inv_freq"] = (10000.0 ** (-torch.arange(n, device="cuda", dtype=torch.float64) / n)).float()
    if case["way"] == "bwd":
        st["dq_out"], st["dk_out"] = rand(b, s, hq, d).to(dt), rand(b, s, hk, d).to(dt)
    return st


def _row_logp(logits, labels):
    """lse and logp of each row, in 64 bits by blocks of rows (input preparation)."""
    lse, logp = [], []
    step = max(1, (1 << 26) // logits.shape[1])
    for at in range(0, logits.shape[0], step):
        z = logits[at:at + step].double() * (1 / TEMPERATURE)
        lse.append(torch.logsumexp(z, 1))
        logp.append(z.gather(1, labels[at:at + step].clamp(min=0)[:, None])[:, 0] - lse[-1])
    return torch.cat(lse), torch.cat(logp)


def _prepare_loss(case, g):
    dt, rows, cols = DTYPES[case["dtype"]], case["rows"], case["cols"]
    rand = lambda *shape: torch.randn(*shape, generator=g, device="cuda")  # noqa: E731
    full = torch.empty(rows, cols + case["pad"], dtype=dt, device="cuda").normal_(0, 3, generator=g)
    logits = full[:, :cols]
    # every other token is the likeliest one, as a sampled policy's often are
    labels = torch.randint(0, cols, (rows,), generator=g, device="cuda")
    labels = torch.where(torch.arange(rows, device="cuda") % 2 == 0, logits.argmax(1), labels)
    lse, logp = _row_logp(logits, labels)
    st = {"case": case, "logits": logits, "labels": labels, "lse": lse.float()}
    st["ref_logp"] = (logp - 0.05 + 0.3 * rand(rows)).float()
    inside = rows - case["tail"]
    left_out = torch.randperm(inside, generator=g, device="cuda")[:case["ignored"]]
    labels[left_out] = IGNORED
    if case["op"] == "policy_loss":
        # log ratios to the sampling policy; none within 1e-3 of a clipping border, where 32 bits would not decide
        ratio = 0.2 * rand(rows)
        for edge in (math.log(1 - CLIP_LOW), math.log(1 + CLIP_HIGH)):
            ratio = torch.where((ratio - edge).abs() < 1e-3, ratio + 3e-3, ratio)
        st["old_logp"] = (logp - ratio).float()
        st["advantages"] = rand(rows)
        st["dloss"] = torch.full((rows,), 1.0 / max(1, rows - case["ignored"]), device="cuda")
        return st
    cuts = torch.randperm(max(1, inside - 1), generator=g, device="cuda")[:2 * case["pairs"] - 1] + 1
    starts = torch.cat([torch.zeros(1, dtype=torch.int64, device="cuda"), cuts.sort().values])
    starts = torch.nn.functional.pad(starts, (0, 2 * case["pairs"] + 1 - starts.numel()), value=inside)
    starts[-1] = inside
    st["seq_starts"] = starts.clamp(max=inside).to(torch.int32)
    if case["way"] == "bwd":
        st["dloss"] = torch.rand(case["pairs"], generator=g, device="cuda") / case["pairs"]
        seq = torch.searchsorted(starts[1:].contiguous(), torch.arange(inside, device="cuda"), right=True)
        part = torch.where(labels[:inside] != IGNORED, logp[:inside] - st["ref_logp"][:inside].double(), 0.0)
        st["log_ratio"] = torch.zeros(2 * case["pairs"], dtype=torch.float64, device="cuda").index_add_(0, seq, part).float()
    return st


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return _prepare_heads(case, g) if case["op"] in ("qk_norm_rope", "rope") else _prepare_loss(case, g)


# ---------------------------------------------------------------- plain forms

def _cos_sin(st):
    """[batch, seq, 1, n] cosines and sines; the angles in 64 bits, where far positions need them."""
    pos = st["positions"].double()
    if st["sections"] is None:
        at = pos.unsqueeze(-1)
    else:
        axis = torch.repeat_interleave(torch.arange(len(st["sections"]), device=pos.device),
                                       torch.tensor(st["sections"], device=pos.device))
        at = pos[axis].movedim(0, -1)
    phi = at * st["inv_freq"].double()
    return phi.cos().float().unsqueeze(-2), phi.sin().float().unsqueeze(-2)


def _rotate(x, cos, sin, interleaved):
    n = cos.shape[-1]
    if interleaved:
        a, b = x[..., 0:2 * n:2], x[..., 1:2 * n:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = x[..., :n], x[..., n:2 * n]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, x[..., 2 * n:]], -1)


def _plain_heads(st):
    case = st["case"]
    cos, sin = _cos_sin(st)
    out, weights = [], []
    for x, w in (("q", "q_weight"), ("k", "k_weight")):
        dt = st[x].dtype
        if case["op"] == "rope":
            out.append(_rotate(st[x].float(), cos, sin, case["interleaved"]).to(dt) if case["way"] == "fwd" else
                       _rotate(st["d" + x + "_out"].float(), cos, -sin, case["interleaved"]).to(dt))
            continue
        v, w = st[x].float(), st[w].float()
        rstd = torch.rsqrt((v * v).mean(-1, keepdim=True) + EPS)
        if case["way"] == "fwd":
            out.append(_rotate(v * rstd * w, cos, sin, case["interleaved"]).to(dt))
            continue
        grad = _rotate(st["d" + x + "_out"].float(), cos, -sin, case["interleaved"])
        unit = v * rstd
        weights.append((grad * unit).sum((0, 1, 2)))
        grad = grad * w
        out.append(((grad - unit * (grad * unit).mean(-1, keepdim=True)) * rstd).to(dt))
    return tuple(out + weights)


def _plain_rows(st):
    """32-bit scaled logits, their lse, logp and which rows count."""
    labels, case = st["labels"], st["case"]
    z = st["logits"].float() * (1 / TEMPERATURE)
    keep = (labels >= 0) & (labels < z.shape[1])
    if case["op"] == "preference_loss":
        keep = keep & (torch.arange(labels.shape[0], device=labels.device) < st["seq_starts"][-1])
    top = z.amax(1, keepdim=True)
    lse = (top + (z - top).exp().sum(1, keepdim=True).log())[:, 0] if case["way"] != "bwd" else st["lse"]
    logp = z.gather(1, labels.clamp(min=0)[:, None])[:, 0] - lse
    return z, torch.where(keep, lse, 0.0), torch.where(keep, logp, 0.0), keep


def _plain_grad(st, z, lse, keep, weight):
    """weight * d logp / d logits, rows left out 0."""
    p = (z - lse[:, None]).exp()
    p.scatter_add_(1, st["labels"].clamp(min=0)[:, None], torch.full_like(lse, -1.0)[:, None])
    grad = p * (weight * (-1 / TEMPERATURE))[:, None]
    return torch.where(keep[:, None], grad, 0.0).to(st["logits"].dtype)


def _plain_policy(st):
    case = st["case"]
    z, lse, logp, keep = _plain_rows(st)
    ratio, adv = (logp - st["old_logp"]).exp(), st["advantages"]
    free, clipped = -ratio * adv, -ratio.clamp(1 - CLIP_LOW, 1 + CLIP_HIGH) * adv
    d = st["ref_logp"] - logp
    kl = torch.where(keep, d.expm1() - d, 0.0)
    loss = torch.where(keep, torch.maximum(free, clipped) + KL_COEF * kl, 0.0)
    if case["way"] == "fwd":
        return loss, logp, lse, kl
    weight = torch.where(clipped > free, 0.0, free) - KL_COEF * d.expm1()
    grad = _plain_grad(st, z, lse, keep, weight * st["dloss"])
    return grad if case["way"] == "bwd" else (loss, logp, lse, kl, grad)


def _plain_preference(st):
    case, starts = st["case"], st["seq_starts"].long()
    pairs = case["pairs"]
    z, lse, logp, keep = _plain_rows(st)
    row = torch.arange(case["rows"], device=z.device)
    seq = torch.searchsorted(starts[1:].contiguous(), row, right=True).clamp(max=2 * pairs - 1)
    if case["way"] == "fwd":
        part = torch.where(keep, logp - st["ref_logp"], 0.0).double()  # a long sum
        log_ratio = torch.zeros(2 * pairs, dtype=torch.float64, device=z.device).index_add_(0, seq, part)
        margin = BETA * (log_ratio[:pairs] - log_ratio[pairs:])
        loss = (1 - SMOOTHING) * _softplus(-margin) + SMOOTHING * _softplus(margin)
        return loss.float(), log_ratio.float(), logp, lse
    margin = BETA * (st["log_ratio"][:pairs] - st["log_ratio"][pairs:])
    up = 1 / (1 + (-margin).exp())
    slope = st["dloss"] * BETA * (SMOOTHING * up - (1 - SMOOTHING) * (1 - up))
    return _plain_grad(st, z, lse, keep, torch.cat([slope, -slope])[seq])


def _softplus(x):
    return x.clamp(min=0) + (-x.abs()).exp().log1p()


# ---------------------------------------------------------------- one pass

def _own_heads(st):
    import dslperfgap_b200 as fw
    case = st["case"]
    how = {"sections": st["sections"], "interleaved": case["interleaved"]}
    at = (st["positions"], st["inv_freq"])
    if case["op"] == "rope":
        if case["way"] == "fwd":
            return fw.rope(st["q"], st["k"], *at, **how)
        return fw.rope_bwd(st["dq_out"], st["dk_out"], *at, **how)
    weights = (st["q_weight"], st["k_weight"])
    if case["way"] == "fwd":
        return fw.qk_norm_rope(st["q"], st["k"], *weights, *at, eps=EPS, **how)
    return fw.qk_norm_rope_bwd(st["dq_out"], st["dk_out"], st["q"], st["k"], *weights, *at, eps=EPS, **how)


def _own_loss(st):
    import dslperfgap_b200 as fw
    case, logits, labels = st["case"], st["logits"], st["labels"]
    how = {"logit_scale": 1 / TEMPERATURE, "ignored_index": IGNORED}
    if case["op"] == "policy_loss":
        how.update(ref_logp=st["ref_logp"], clip_low=CLIP_LOW, clip_high=CLIP_HIGH, kl_coef=KL_COEF)
        rows = (st["old_logp"], st["advantages"])
        if case["way"] == "fwd":
            return fw.policy_loss_fwd(logits, labels, *rows, **how)
        if case["way"] == "bwd":
            return fw.policy_loss_bwd(st["dloss"], logits, st["lse"], labels, *rows, **how)
        return fw.policy_loss_fwd_bwd(logits, labels, *rows, st["dloss"], **how)
    how.update(beta=BETA, smoothing=SMOOTHING)
    if case["way"] == "fwd":
        return fw.preference_loss_fwd(logits, labels, st["seq_starts"], st["ref_logp"], **how)
    return fw.preference_loss_bwd(st["dloss"], logits, st["lse"], labels, st["seq_starts"], st["log_ratio"], **how)


def run(state):
    op = state["case"]["op"]
    if own:
        return _own_heads(state) if op in ("qk_norm_rope", "rope") else _own_loss(state)
    if op in ("qk_norm_rope", "rope"):
        return _plain_heads(state)
    return _plain_policy(state) if op == "policy_loss" else _plain_preference(state)


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] in ("qk_norm_rope", "rope"):
        tokens = case["batch"] * case["seq"]
        values = tokens * (case["hq"] + case["hk"]) * case["dim"]
        passes = 3 if case["op"] == "qk_norm_rope" and case["way"] == "bwd" else 2
        once = 8 * tokens * case["axes"] + 2 * case["rot"]
        if case["op"] == "qk_norm_rope":  # the weights, and in the backward pass their gradients
            once += 2 * case["dim"] * (size + (4 if case["way"] == "bwd" else 0))
        return {"bytes": passes * values * size + once, "flops": 12 * values}
    rows, cols = case["rows"], case["cols"]
    read = (rows - case["ignored"] - case["tail"]) * cols
    written = rows * cols if case["way"] != "fwd" else 0
    policy = case["op"] == "policy_loss"
    per_row = 8 + {"fwd": 28 if policy else 12, "bwd": 20 if policy else 4, "fwd_bwd": 32}[case["way"]]
    return {"bytes": (read + written) * size + rows * per_row + 32 * case["pairs"], "flops": 4 * read + 4 * written}


# ---------------------------------------------------------------- 64 bits

def _exact_turn(x, st):
    """The rotation as a complex product."""
    case = st["case"]
    n = case["rot"] // 2
    pos = st["positions"].double()
    if st["sections"] is None:
        pos = pos.unsqueeze(0)
    bounds = st["sections"] or (n,)
    phi = torch.cat([p.unsqueeze(-1) * f for p, f in zip(pos, st["inv_freq"].double().split(list(bounds)))], -1)
    unit = torch.polar(torch.ones_like(phi), phi).unsqueeze(-2)
    if case["interleaved"]:
        z = torch.view_as_complex(x[..., :2 * n].unflatten(-1, (n, 2)).contiguous()) * unit
        y = torch.view_as_real(z).flatten(-2)
    else:
        z = torch.complex(x[..., :n].contiguous(), x[..., n:2 * n].contiguous()) * unit
        y = torch.cat([z.real, z.imag], -1)
    return torch.cat([y, x[..., 2 * n:]], -1)


def _exact_heads(st):
    case = st["case"]
    out, weights = [], []
    for name in ("q", "k"):
        x = st[name].double().requires_grad_(case["way"] == "bwd")
        w = st[name + "_weight"].double().requires_grad_(case["way"] == "bwd")
        with torch.set_grad_enabled(case["way"] == "bwd"):
            v = x if case["op"] == "rope" else x / (x.square().mean(-1, keepdim=True) + EPS).sqrt() * w
            y = _exact_turn(v, st)
            if case["way"] == "fwd":
                out.append(y)
            elif case["op"] == "rope":
                out += torch.autograd.grad(y, [x], st["d" + name + "_out"].double())
            else:
                dx, dw = torch.autograd.grad(y, [x, w], st["d" + name + "_out"].double())
                out.append(dx)
                weights.append(dw)
    return tuple(out + weights)


def _exact_loss(st):
    case, labels = st["case"], st["labels"]
    bwd = case["way"] != "fwd"
    rows = labels.shape[0]
    used = labels >= 0
    if case["op"] == "preference_loss":
        used = used & (torch.arange(rows, device="cuda") < rows - case["tail"])
    used = used.nonzero()[:, 0]
    x = st["logits"][used].double().requires_grad_(bwd)
    whole = lambda v: torch.zeros(rows, dtype=torch.float64, device="cuda").index_copy(0, used, v)  # noqa: E731
    with torch.set_grad_enabled(bwd):
        table = torch.log_softmax(x / TEMPERATURE, 1)
        logp = table[torch.arange(used.numel(), device="cuda"), labels[used]]
        if case["op"] == "policy_loss":
            ratio, adv = torch.exp(logp - st["old_logp"][used].double()), st["advantages"][used].double()
            d = st["ref_logp"][used].double() - logp
            kl = torch.exp(d) - d - 1
            loss = -torch.min(ratio * adv, ratio.clamp(1 - CLIP_LOW, 1 + CLIP_HIGH) * adv) + KL_COEF * kl
            total = (loss * st["dloss"][used].double()).sum() if bwd else None
        else:
            first = st["seq_starts"].tolist()
            part = logp - st["ref_logp"][used].double()
            where = torch.bucketize(used, torch.tensor(first[1:], device="cuda"), right=True)
            log_ratio = torch.stack([part[where == s].sum() for s in range(2 * case["pairs"])])
            margin = BETA * (log_ratio[:case["pairs"]] - log_ratio[case["pairs"]:])
            loss = -(1 - SMOOTHING) * torch.nn.functional.logsigmoid(margin) - SMOOTHING * torch.nn.functional.logsigmoid(-margin)
            total = (loss * st["dloss"].double()).sum() if bwd else None
    grad = None
    if bwd:
        grad = torch.zeros(rows, case["cols"], dtype=torch.float64, device="cuda")
        grad[used] = torch.autograd.grad(total, [x])[0]
    if case["way"] == "bwd":
        return grad
    lse = whole((x.detach()[:, 0] / TEMPERATURE - table.detach()[:, 0]))
    if case["op"] == "policy_loss":
        out = (whole(loss.detach()), whole(logp.detach()), lse, whole(kl.detach()))
        return out + (grad,) if bwd else out
    return loss, log_ratio, whole(logp), lse


def exact(case, seed):
    st = prepare(case, seed)
    return _exact_heads(st) if case["op"] in ("qk_norm_rope", "rope") else _exact_loss(st)
