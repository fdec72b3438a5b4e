"""rope and qk_norm_rope, forward and backward, against a plain 64-bit
evaluation: types, head sizes with and without vector access, partial and
interleaved rotation, position axes, far and negative positions, strided and
broadcast inputs, one token to thousands, empty inputs, graphs, streams and
repeatability."""
import pytest
import torch

import dslperfgap_b200 as B
import heads_ref as R
from dslperfgap_b200 import _lib

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-6
#: a lane's few rows, then 5 lane steps, 8 warps, 148 + 8 CTAs one after another
DW_STEPS = 256


def make(tokens, hq, hk, d, rot, dt, seed=0, axes=0, far=0, wdt=None):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    q, k = rn(*tokens, hq, d).to(DT[dt]), rn(*tokens, hk, d).to(DT[dt])
    qw, kw = ((1 + 0.2 * rn(d)).to(DT[wdt or dt]) for _ in range(2))
    n = rot // 2
    freq = (10000.0 ** (-torch.arange(n, device="cuda", dtype=torch.float64) / n)).float()
    shape = ((axes,) if axes else ()) + tuple(tokens)
    pos = torch.randint(-50, 5000, shape, generator=g, device="cuda") + far
    sections = None
    if axes:
        cuts = [n // (axes + 1)] * (axes - 1)
        sections = (n - sum(cuts), *cuts)
    return q, k, qw, kw, pos, freq, sections


def check_all(tokens, hq, hk, d, rot, dt, inter=False, axes=0, far=0, wdt=None, seed=0):
    q, k, qw, kw, pos, freq, sec = make(tokens, hq, hk, d, rot, dt, seed, axes, far, wdt)
    phi = R.angles(pos, freq, sec, tokens)
    how = dict(sections=sec, interleaved=inter)
    for got, x in zip(B.rope(q, k, pos, freq, **how), (q, k)):
        assert got.shape == x.shape and got.dtype == x.dtype and got.is_contiguous()
        R.check_forward(got, x, None, phi, inter, EPS, "rope")
    for got, x in zip(B.rope_bwd(q, k, pos, freq, **how), (q, k)):
        R.check_forward(got, x, None, -phi, inter, EPS, "rope_bwd")
    for got, x, w in zip(B.qk_norm_rope(q, k, qw, kw, pos, freq, eps=EPS, **how), (q, k), (qw, kw)):
        R.check_forward(got, x, w, phi, inter, EPS, "qk_norm_rope")
    dq, dk = torch.randn_like(q), torch.randn_like(k)
    out = B.qk_norm_rope_bwd(dq, dk, q, k, qw, kw, pos, freq, eps=EPS, **how)
    check_backward(out, dq, dk, q, k, qw, kw, phi, inter)


def check_backward(out, dq, dk, q, k, qw, kw, phi, inter):
    for i, (dy, x, w) in enumerate(((dq, q, qw), (dk, k, kw))):
        dx, dw, slack, terms = R.backward(dy, x, w, phi, inter, EPS)
        assert out[i].shape == x.shape and out[i].dtype == x.dtype and out[2 + i].dtype == torch.float32
        R.close(out[i], dx, slack, f"dx[{i}]")
        R.close(out[2 + i], dw, (DW_STEPS * R.U + R.BWD) * terms, f"dw[{i}]")


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("d,rot", [(128, 128), (64, 64), (256, 256), (80, 40), (72, 72), (96, 96), (128, 32), (576, 64),
                                   (40, 8), (36, 20), (5, 4), (2, 2), (33, 32), (1024, 1024), (72, 36), (200, 100), (8, 4), (16, 12)])
def test_head_sizes(d, rot, inter, dt):
    check_all((7, 9), 5, 2, d, rot, dt, inter)


@pytest.mark.parametrize("tokens", [(1,), (2,), (1, 1), (3, 1), (1, 150), (4099,), (3, 1111)])
@pytest.mark.parametrize("hq,hk", [(1, 1), (8, 1), (12, 3), (32, 8), (3, 7)])
def test_lengths_and_heads(tokens, hq, hk):
    check_all(tokens, hq, hk, 128, 128, "bf16")


@pytest.mark.parametrize("path", ["stream"])
@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("inter", [False, True])
def test_scalar_path(path, dt, inter):
    with _lib.kernel_path(path):
        check_all((3, 70), 4, 2, 128, 64, dt, inter, axes=2)


@pytest.mark.parametrize("axes", [1, 2, 3, 4])
@pytest.mark.parametrize("inter", [False, True])
def test_axes(axes, inter):
    check_all((2, 301), 4, 2, 128, 128, "bf16", inter, axes=axes)
    check_all((77,), 4, 2, 72, 72, "f32", inter, axes=axes)


def test_empty_sections_of_axes():
    q, k, _, _, _, freq, _ = make((9,), 2, 1, 64, 64, "f32")
    pos = torch.arange(27, device="cuda").view(3, 9)
    for sec in ((32, 0, 0), (0, 0, 32), (0, 32, 0)):
        got = B.rope(q, k, pos, freq, sections=sec)
        phi = R.angles(pos[sec.index(32)], freq, None, (9,))
        R.check_forward(got[0], q, None, phi, False, EPS)


@pytest.mark.parametrize("far", [131071, 1 << 20, (1 << 31) + 12345, -(1 << 24)])
def test_far_positions(far):
    check_all((50,), 4, 4, 64, 64, "f32", far=far)


@pytest.mark.parametrize("wdt", ["f32", "f16", "bf16"])
def test_weight_types(wdt):
    check_all((33,), 4, 2, 128, 128, "bf16", wdt=wdt)


def test_int32_and_broadcast_positions():
    q, k, qw, kw, _, freq, _ = make((5, 40), 4, 2, 128, 128, "bf16")
    pos = torch.arange(40, device="cuda", dtype=torch.int32) + 7
    full = pos.long().expand(5, 40).contiguous()
    want = B.qk_norm_rope(q, k, qw, kw, full, freq)
    for p in (pos, pos.view(1, 40), pos.expand(5, 40)):
        got = B.qk_norm_rope(q, k, qw, kw, p, freq)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    got = B.qk_norm_rope(q, k, qw, kw, pos.expand(1, 5, 40), freq, sections=(64,))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    one = B.rope(q, k, torch.tensor(3, device="cuda"), freq)
    R.check_forward(one[0], q, None, R.angles(torch.tensor(3, device="cuda"), freq, None, (5, 40)), False, EPS)


def views(kind):
    """q [3, 50, 6, 64] and k [3, 50, 2, 64] as views of one kind."""
    g = torch.Generator(device="cuda").manual_seed(3)
    if kind == "fused":
        x = torch.randn(3, 50, 10 * 64, generator=g, device="cuda").bfloat16()
        return x[..., :6 * 64].unflatten(-1, (6, 64)), x[..., 6 * 64:8 * 64].unflatten(-1, (2, 64))
    if kind == "heads_first":
        x = torch.randn(3, 8, 50, 64, generator=g, device="cuda").bfloat16()
        return x[:, :6].transpose(1, 2), x[:, 6:].transpose(1, 2)
    if kind == "odd_offset":
        x = torch.randn(3, 50, 8 * 64 + 3, generator=g, device="cuda").bfloat16()
        return x[..., 1:1 + 6 * 64].unflatten(-1, (6, 64)), x[..., 3 + 6 * 64:].unflatten(-1, (2, 64))
    if kind == "broadcast":
        x = torch.randn(1, 50, 1, 64, generator=g, device="cuda").bfloat16()
        return x.expand(3, 50, 6, 64), x.expand(3, 50, 2, 64)
    x = torch.randn(3, 50, 8, 64, 2, generator=g, device="cuda").bfloat16()  # strided features
    return x[:, :, :6, :, 0], x[:, :, 6:, :, 1]


@pytest.mark.parametrize("kind", ["fused", "heads_first", "odd_offset", "broadcast", "strided_features"])
def test_views_equal_dense(kind):
    q, k = views(kind)
    _, _, qw, kw, pos, freq, _ = make((3, 50), 6, 2, 64, 64, "bf16")
    dense = q.contiguous(), k.contiguous()
    phi = R.angles(pos, freq, None, (3, 50))
    for got, x, w in zip(B.qk_norm_rope(q, k, qw, kw, pos, freq), dense, (qw, kw)):
        assert got.is_contiguous()
        R.check_forward(got, x, w, phi, False, EPS, kind)
    dq, dk = torch.randn_like(dense[0]), torch.randn_like(dense[1])
    check_backward(B.qk_norm_rope_bwd(dq, dk, q, k, qw, kw, pos, freq), dq, dk, *dense, qw, kw, phi, False)
    check_backward(B.qk_norm_rope_bwd(q, k, dq, dk, qw, kw, pos, freq), *dense, dq, dk, qw, kw, phi, False)
    for got, x in zip(B.rope_bwd(q, k, pos, freq), dense):
        R.check_forward(got, x, None, -phi, False, EPS, kind)


def test_empty():
    _, _, qw, kw, _, freq, _ = make((1,), 1, 1, 64, 64, "bf16")
    none = torch.empty(0, 4, 64, device="cuda", dtype=torch.bfloat16)
    pos = torch.empty(0, dtype=torch.long, device="cuda")
    assert [t.shape for t in B.qk_norm_rope(none, none, qw, kw, pos, freq)] == [none.shape] * 2
    dq, dk, dqw, dkw = B.qk_norm_rope_bwd(none, none, none, none, qw, kw, pos, freq)
    assert dq.shape == none.shape and not dqw.any() and not dkw.any()
    # k without heads: q is worked on, k's weight gradient is 0
    q, _, qw, kw, pos, freq, _ = make((11,), 4, 1, 64, 64, "bf16")
    k0 = q[:, :0]
    phi = R.angles(pos, freq, None, (11,))
    got = B.qk_norm_rope(q, k0, qw, kw, pos, freq)
    R.check_forward(got[0], q, qw, phi, False, EPS)
    got = B.qk_norm_rope(k0, q, qw, kw, pos, freq)
    R.check_forward(got[1], q, kw, phi, False, EPS)
    out = B.qk_norm_rope_bwd(q, k0, q, k0, qw, kw, pos, freq)
    dx, dw, slack, terms = R.backward(q, q, qw, phi, False, EPS)
    R.close(out[0], dx, slack)
    R.close(out[2], dw, (DW_STEPS * R.U + R.BWD) * terms)
    assert not out[3].any()
    out = B.qk_norm_rope_bwd(k0, q, k0, q, qw, kw, pos, freq)
    assert not out[2].any() and out[3].any()


def test_zero_rows_and_special_values():
    """A row of zeros stays zero and finite (eps), NaN and inf stay in their own row."""
    q, k, qw, kw, pos, freq, _ = make((6,), 2, 2, 64, 64, "f32")
    q[1], q[2, 0, 3], q[3, 1, 5] = 0, float("nan"), float("inf")
    yq, _ = B.qk_norm_rope(q, k, qw, kw, pos, freq)
    assert not yq[1].any()
    assert yq[2, 0].isnan().all() and not yq[2, 1].isnan().any()
    assert yq[3, 1].isnan().any() and not yq[3, 0].isnan().any()
    assert yq[[0, 4, 5]].isfinite().all()


def test_gradient_against_differences():
    """The backward pass against central differences of the 64-bit forward."""
    q, k, qw, kw, pos, freq, _ = make((3,), 2, 1, 16, 12, "f32")
    dq, dk = torch.randn_like(q), torch.randn_like(k)
    out = B.qk_norm_rope_bwd(dq, dk, q, k, qw, kw, pos, freq)
    phi = R.angles(pos, freq, None, (3,))
    f = lambda x, w: (R.turn(R.norm(x, w, EPS)[0], phi, False) * dq.double()).sum()  # noqa: E731
    x, w, h = q.double(), qw.double(), 1e-5
    for i in range(0, x.numel(), 7):
        e = torch.zeros_like(x).view(-1)
        e[i] = h
        slope = (f(x + e.view_as(x), w) - f(x - e.view_as(x), w)) / (2 * h)
        # third derivatives of order 10 times h^2, and 64 half steps of terms of order 10
        assert abs(out[0].view(-1)[i].item() - slope.item()) < 1e-8 + 640 * R.U
    for i in range(16):
        e = torch.zeros_like(w)
        e[i] = h
        slope = (f(x, w + e) - f(x, w - e)) / (2 * h)
        assert abs(out[2][i].item() - slope.item()) < 1e-8 + 640 * R.U


def test_same_bits_every_time():
    q, k, qw, kw, pos, freq, _ = make((2, 777), 8, 8, 64, 64, "bf16")
    a = B.qk_norm_rope_bwd(q, k, q, k, qw, kw, pos, freq)
    for _ in range(3):
        b = B.qk_norm_rope_bwd(q, k, q, k, qw, kw, pos, freq)
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_graph_and_other_stream():
    q, k, qw, kw, pos, freq, _ = make((64,), 8, 2, 128, 128, "bf16")
    run = lambda: B.qk_norm_rope(q, k, qw, kw, pos, freq) + B.qk_norm_rope_bwd(q, k, q, k, qw, kw, pos, freq)  # noqa: E731
    run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = run()
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):  # two graphs alive at once
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(run())
    q.copy_(torch.randn_like(q))
    pos.add_(100)
    want = run()
    for g in graphs:
        g.replay()
    torch.cuda.synchronize()
    for out in outs:
        assert all(torch.equal(a, b) for a, b in zip(out, want))
    assert not torch.equal(on_side[0], want[0])


def test_fast_path_equals_python_path(monkeypatch):
    import importlib
    q, k, qw, kw, pos, freq, sec = make((3, 70), 8, 2, 128, 128, "bf16", axes=3)
    calls = [("rope", "rope", (q, k, pos, freq, sec)), ("rope", "rope_bwd", (q, k, pos, freq, sec, True)),
             ("qk_norm_rope", "qk_norm_rope", (q, k, qw, kw, pos, freq, 1e-5, sec)),
             ("qk_norm_rope", "qk_norm_rope_bwd", (q, k, q, k, qw, kw, pos, freq, 1e-5, sec)),
             ("rope", "rope", (q[0], k[0], pos[:, 0], freq, list(sec)))]
    for module, name, args in calls:
        mod = importlib.import_module(f"dslperfgap_b200.{module}.cuda_impl")
        assert _lib.torch_ops() is not None
        fast = getattr(mod, name)(*args)
        with monkeypatch.context() as m:
            m.setattr(mod, f"_fast_{name}", lambda *a: None)
            slow = getattr(mod, name)(*args)
        assert len(fast) == len(slow) and all(torch.equal(a, b) for a, b in zip(fast, slow)), name


def test_guard_bytes_around_outputs():
    """The C entry writes its outputs and nothing beside them."""
    import ctypes
    from dslperfgap_b200 import _heads
    for d, rot in ((128, 128), (72, 36), (33, 32)):
        q, k, qw, kw, pos, freq, _ = make((13,), 3, 2, d, rot, "bf16")
        pos, freq, h = _heads.layout(q, k, pos, freq, None, False, "t", q, k, qw)
        sizes = [q.numel() * 2, k.numel() * 2, d * 4, d * 4]
        need = ctypes.c_int64(0)
        _lib.check(_lib.load().dslpg_qk_norm_rope_bwd_workspace_bytes(d, ctypes.byref(need)), "ws")
        sizes.append(need.value)
        bufs = [torch.full((s + 512,), 0xA5, dtype=torch.uint8, device="cuda") for s in sizes]
        at = [b.data_ptr() + 256 for b in bufs]
        _lib.launch(q.device, "dslpg_qk_norm_rope_bwd", q.data_ptr(), k.data_ptr(), q.data_ptr(), k.data_ptr(),
                    qw.data_ptr(), kw.data_ptr(), pos.data_ptr(), freq.data_ptr(), *at[:4], ctypes.addressof(h), EPS,
                    at[4], need.value)
        torch.cuda.synchronize()
        for b in bufs:
            assert (b[:256] == 0xA5).all() and (b[-256:] == 0xA5).all()
        want = B.qk_norm_rope_bwd(q, k, q, k, qw, kw, pos, freq, eps=EPS)
        assert torch.equal(bufs[0][256:-256], want[0].view(-1).view(torch.uint8))


@pytest.mark.parametrize("axes", [1, 4])
@pytest.mark.parametrize("hq,hk,d,dt", [(1, 1, 64, "bf16"), (4, 1, 96, "f16"), (1, 4, 72, "f32")])
def test_few_heads_many_tokens(hq, hk, d, dt, axes):
    """Tiles of 8 tokens, several of a tile in one copy where they follow one another, and not where a sequence ends
    (an odd length) or the batches lie apart: the same bits each way."""
    check_all((2, 5003), hq, hk, d, d, dt, axes=axes)
    q, k, qw, kw, pos, freq, sec = make((2, 5003), hq, hk, d, d, dt, axes=axes)
    apart = [torch.zeros(2, 5010, *x.shape[2:], dtype=x.dtype, device="cuda") for x in (q, k)]
    for a, x in zip(apart, (q, k)):
        a[:, :5003] = x
    q2, k2 = (a[:, :5003] for a in apart)
    ways = [(q, k), (q2, k2), (q, k2)]
    for f in (lambda a, b: B.qk_norm_rope(a, b, qw, kw, pos, freq, sections=sec),
              lambda a, b: B.rope(a, b, pos, freq, sections=sec),
              lambda a, b: B.qk_norm_rope_bwd(q, k, a, b, qw, kw, pos, freq, sections=sec)):
        first = f(*ways[0])
        for way in ways[1:]:
            assert all(torch.equal(g, w) for g, w in zip(f(*way), first))
