// heads.cu — per-head RMSNorm with the rotary position rotation, and the
// rotation alone, forward and backward (sm_100a).
//
// A row is one head of one token: x[0..D). With n = R/2 frequencies f_i, a(i)
// the position axis of frequency i and phi_i = pos[a(i)] * f_i:
//   rstd = 1 / sqrt(mean(x^2) + eps);  u = x * rstd * w   (rotation alone: u = x)
//   (y_i, y_j) = (u_i cos phi - u_j sin phi, u_j cos phi + u_i sin phi),
//   (i, j) = (i, i + n), or (2i, 2i + 1) interleaved;  y_d = u_d for d >= R.
// Backward: g = dy rotated by -phi, c = sum(g w x),
//   dx = rstd * (w g - x rstd^2 c / D);  dw = sum over rows of g x rstd.
// The rotation's own backward is the rotation by -phi.
//
// Angles: as fractions of a turn in 64-bit fixed point, where f_i / 2 pi times an
// integer position is one wrapping integer product: the whole turns fall off
// exactly, for negative and far positions alike. f_i / 2 pi is right to its last
// bit for |f_i| up to 2^18, so an angle is off by |position| 2^-64 turns beside its
// own rounding, and the cosine keeps its 32-bit accuracy for positions up to 2^38.
// (A further 32 bits, for tiles that hold a position beyond 32 bits alone, would
// reach every int64 position, but the test for such tiles took 3 to 7 % of tokens
// of few heads; the whole in double precision took 0.9 us a token in its warp, a
// chain of conversions and roundings.) The n angles of a token are formed once and
// serve all of its heads.
//
// Lanes: a row is cut into units of two V-element vectors that hold both
// members of V rotated pairs (vectors u and u + n/V; interleaved 2u and
// 2u + 1), so the rotation needs no exchange between lanes; the features
// past R are units of two neighbouring vectors. A lane takes one unit, a warp
// takes 32 / units rows (a group) at a time.
//
// Pipeline: a CTA walks tiles of a few whole tokens (or of some heads of one).
// Warp 0 copies a tile's rows into a ring of shared-memory stages with
// cp.async.bulk, the next warps form its tokens' angles there, and the other
// warps turn rows into outputs. Rows lie in a stage as in the output, tensor by
// tensor, so a row's place in both is its number, and a group may span tokens.
// Before this, each warp copied its own rows (cp.async, one lane a vector) and
// formed its own angles; the addresses, bounds and waits of that took 200 of 440
// instructions a group of rows: forward 61.0 us against 59.5 for 16384 tokens of
// 32 + 8 heads of 128 in bf16 (a torch copy of the same bytes: 58), backward 108
// against 90, the rotation of 29971 tokens of 16 + 16 heads 86.8 against 82
// (81.5), and one decoded token 6.2 against 4.2.
#include <algorithm>

#include "common.cuh"
#include "pipe.cuh"

namespace dslpg {

// Waits that ran out of time in this file's kernels.
static __device__ unsigned int g_heads_timeouts;

struct HeadArgs {
  const void* x[2];    // q, k: the rows (rotation backward: dy)
  const void* dy[2];   // norm backward: the gradients of the outputs
  void* y[2];          // outputs, dense [tokens, heads, D]
  const void* w[2];    // [D] weights
  const void* pos;
  const float* inv_freq;
  float* partial;      // norm backward: [CTAs][2][D] sums for dw
  int64_t xs[2][3];    // batch, sequence and head strides of x
  int64_t dys[2][3];
  int64_t ps[3];       // axis, batch and sequence strides of pos
  uint32_t tokens, seq;
  int heads[2];
  int D, n;            // features; rotated pairs
  int bound[3];        // first frequency of axes 1, 2, 3
  int axes;
  int rot_units, units, rpw;  // rpw: rows of a group, 32 / units
  // Tiles: tt tokens with all their heads, or (parts > 1) one token and `part` of its heads.
  int tt, part, parts;
  uint32_t tiles;
  int stages, stage_bytes, row_bytes;
  int angle_warps, row_warps;
  int pairs;           // an angle warp forms two tokens' angles side by side
  int groups;          // groups of a tile: those of q's rows, then those of k's (the last ones may be empty)
  int q_groups, q_warps;  // norm backward: groups of q's rows in every tile, and the row warps that take them
  // From a tile of a CTA to its next one (parts == 1): tokens modulo seq; what is
  // added to a token's place in x, dy and pos, and once more where a sequence ends.
  uint32_t s_step;
  int64_t x_step[2], x_carry[2], dy_step[2], dy_carry[2], p_step, p_carry;
  uint32_t magic[2];   // r / heads of a token in the tile = umulhi(r, magic); 0: r itself
  int wdt, pos64, interleaved;
  float eps, inv_d, sign;
};

enum HeadOp : int { kRotate, kNorm, kNormBwd };

// V elements of T.
template <typename T, int V> struct Pack {
  static constexpr int kBytes = V * static_cast<int>(sizeof(T));
  static_assert(kBytes == 4 || kBytes == 8 || kBytes == 16, "4-, 8- or 16-byte vectors");
};

// Plain float32 arithmetic throughout: packed pairs (fma.f32x2) took more
// instructions here (48 M against 41 M for a rotation of 29971 tokens of 32
// heads), as their operands have to be moved into register pairs.
template <typename T, int V> DSLPG_DEV void lds_vec(uint32_t at, float (&f)[V]) {
  Vec16 v{{0u, 0u, 0u, 0u}};
  if constexpr (Pack<T, V>::kBytes == 16) v = lds16(at);
  else if constexpr (Pack<T, V>::kBytes == 4) asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v.w[0]) : "r"(at) : "memory");
  else asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.w[0]), "=r"(v.w[1]) : "r"(at) : "memory");
  float all[Elt<T>::kPerVec];
  unpack<T>(v, all);
#pragma unroll
  for (int i = 0; i < V; ++i) f[i] = all[i];
}

template <typename T, int V> DSLPG_DEV void st_vec(T* dst, const float (&f)[V]) {
  if constexpr (sizeof(T) == 4 && V == 2) st_stream8(dst, __float_as_uint(f[0]), __float_as_uint(f[1]));
  else if constexpr (V == 2) asm volatile("st.global.u32 [%0], %1;" ::"l"(dst), "r"(pack2<T>(f[0], f[1])) : "memory");
  else StoreOut<T, V>::run(dst, f);
}

// The part of a turn that one position step makes, in units of 2^-64 turns, rounded to the nearest. 1 / (2 pi) is taken
// in two parts, as one double's rounding (2^-55 |f| turns) shows at positions of 2^31: the first has 29 bits, so that
// its product with a float32 is exact, the second's is off by less than 2^-83 |f|.
DSLPG_DEV uint64_t turn_per_step(float f) {
  const double size = fabs(static_cast<double>(f));
  auto fraction = [](double turns) { return (turns - floor(turns)) * 0x1p64; };
  const double a = fraction(size * 0x1.45f306dp-3), b = fraction(size * 0x1.9391054a7f09dp-32);
  const uint64_t whole_a = static_cast<uint64_t>(a), whole_b = static_cast<uint64_t>(b);
  const double rest = (a - static_cast<double>(whole_a)) + (b - static_cast<double>(whole_b));
  const uint64_t step = whole_a + whole_b + static_cast<uint64_t>(rest + 0.5);
  return f < 0.f ? 0 - step : step;
}

// Cosine and sine (times `sign`) of position p at a frequency's turn_per_step.
// For 16-bit rows the SFU's, a fifth of the instructions: off by at most 2^-19.9 (2^-21.2 its own on -pi .. pi, and the
// argument's three roundings of pi 2^-24), far inside the rows' own rounding (2^-12, 2^-9).
template <bool EXACT> DSLPG_DEV float2 angle_of(int64_t p, uint64_t step, float sign) {
  const int turn = static_cast<int>((static_cast<uint64_t>(p) * step) >> 32);  // 2^-32 turns, -2^31 .. 2^31
  float sn, cn;
  if constexpr (EXACT) {
    sincospif(static_cast<float>(turn) * 0x1p-31f, &sn, &cn);
  } else {
    const float a = static_cast<float>(turn) * 1.4629180793e-9f;  // 2 pi / 2^32
    sn = __sinf(a);
    cn = __cosf(a);
  }
  return make_float2(cn, sn * sign);
}

DSLPG_DEV int axis_of(const HeadArgs& a, int i) {
  return i >= a.n ? 0 : (i >= a.bound[0]) + (i >= a.bound[1]) + (i >= a.bound[2]);
}

// The positions of the token at `at` in pos: each of the first lanes reads one axis'.
DSLPG_DEV int64_t lane_position(const HeadArgs& a, int64_t at, int lane) {
  if (lane >= a.axes) return 0;
  const int64_t j = at + lane * a.ps[0];
  return a.pos64 ? static_cast<const int64_t*>(a.pos)[j] : static_cast<const int32_t*>(a.pos)[j];
}

// Angles of a token for this warp, cs[i] = (cos, sin) of frequency i, from its lanes' positions.
template <bool EXACT> DSLPG_DEV void fill_angles(const HeadArgs& a, const uint64_t* freq, float2* cs, int64_t p, int lane) {
  __syncwarp();
  for (int i0 = 0; i0 < a.n; i0 += 32) {
    const int i = i0 + lane;
    const int64_t mine = __shfl_sync(0xffffffffu, static_cast<long long>(p), axis_of(a, i));
    if (i < a.n) cs[i] = angle_of<EXACT>(mine, freq[i], a.sign);
  }
  __syncwarp();
}

// Vector indexes of unit u's two vectors.
template <bool INTER>
DSLPG_DEV void unit_vectors(const HeadArgs& a, int u, int& ia, int& ib) {
  const bool half = u < a.rot_units && !INTER;
  ia = half ? u : 2 * u;  // past the rotated ones: 2 rot_units + 2 (u - rot_units)
  ib = half ? u + a.rot_units : 2 * u + 1;
}

// Sums over the `units` lanes of a row, in all of them.
template <int K> DSLPG_DEV void row_sums(float (&v)[K], int units, int u, int lane) {
  auto swap = [&](int o) {
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
  };
  if (units == 8) {  // 128 features of 16 bits, 64 of 32 bits
    swap(1);
    swap(2);
    swap(4);
  } else if ((units & (units - 1)) == 0) {
    for (int o = 1; o < units; o <<= 1) swap(o);
  } else {
    for (int o = 1; o < units; o <<= 1) {  // lane u holds the sum of u .. u + 2 o - 1 inside the row
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const float t = __shfl_down_sync(0xffffffffu, v[k], o);
        if (u + o < units) v[k] += t;
      }
    }
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] = __shfl_sync(0xffffffffu, v[k], lane - u);
  }
}

// What a lane does in the tile kernel.
template <bool INTER> struct Lane {
  int u, sub, ia, ib;
  bool active;
  DSLPG_DEV Lane(const HeadArgs& a, int lane) {
    sub = lane / a.units;
    u = lane - sub * a.units;
    active = sub < a.rpw;
    unit_vectors<INTER>(a, u, ia, ib);
  }
};

// Tables that a lane reads as its unit's values, four at a time: planes of
// float4, plane j holding values 4j .. 4j + 3 of every unit (or vector), so that
// neighbouring lanes read neighbouring 16 bytes.
//   angles: (cos, sin) of two frequencies in a plane entry, V / 2 planes;
//   weights: V / 4 planes (one of float2 when V is 2).
template <int V> DSLPG_DEV int angle_slot(int i, int rot_units) {  // float2 index of frequency i
  const int u = i / V, e = i - u * V;
  return ((e >> 1) * rot_units + u) * 2 + (e & 1);
}
template <int V> DSLPG_DEV int weight_slot(int d, int vecs) {  // float index of feature d
  constexpr int P = V < 4 ? V : 4;
  const int v = d / V, e = d - v * V;
  return ((e / P) * vecs + v) * P + e % P;
}

template <int V> DSLPG_DEV void read_weights(const float* w, int vec, int vecs, float (&f)[V]) {
  if constexpr (V >= 4) {
#pragma unroll
    for (int j = 0; j < V / 4; ++j) {
      const float4 q = reinterpret_cast<const float4*>(w)[j * vecs + vec];
      f[4 * j] = q.x;
      f[4 * j + 1] = q.y;
      f[4 * j + 2] = q.z;
      f[4 * j + 3] = q.w;
    }
  } else {
    const float2 q = reinterpret_cast<const float2*>(w)[vec];
    f[0] = q.x;
    f[1] = q.y;
  }
}

// Rotate a unit's V pairs in place: half-split (x0 in fa, x1 in fb), or
// interleaved (2e, 2e + 1 of fa, then of fb).
template <int V, bool INTER>
DSLPG_DEV void turn(float (&fa)[V], float (&fb)[V], const float4* angles, int rot_units) {
#pragma unroll
  for (int j = 0; j < V / 2; ++j) {
    const float4 cs = angles[j * rot_units];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int e = 2 * j + k;
      float& x0 = INTER ? (e < V / 2 ? fa[(2 * e) % V] : fb[(2 * e) % V]) : fa[e];
      float& x1 = INTER ? (e < V / 2 ? fa[(2 * e) % V + 1] : fb[(2 * e) % V + 1]) : fb[e];
      const float c = k ? cs.z : cs.x, s = k ? cs.w : cs.y;
      const float y0 = x0 * c - x1 * s;
      x1 = x1 * c + x0 * s;
      x0 = y0;
    }
  }
}

// Parts of a CTA's dynamic shared memory, in this order.
struct HeadSmem {
  int stages, stage_bytes, angle_bytes, n, weight_floats, sum_bytes;
  __host__ __device__ int angles() const { return stages * stage_bytes; }            // [stages][tt][planes]
  __host__ __device__ int freq() const { return angles() + stages * angle_bytes; }   // uint64 [n]
  __host__ __device__ int weight() const { return (freq() + 8 * n + 15) & ~15; }     // [2][weight_floats]
  __host__ __device__ int sums() const { return weight() + 8 * weight_floats; }      // [row warps][D] floats
  __host__ __device__ int bars() const { return sums() + sum_bytes; }
  __host__ __device__ int total() const { return bars() + 16 * stages; }
};

__host__ __device__ inline HeadSmem head_smem(const HeadArgs& a, int op) {
  return HeadSmem{a.stages, a.stage_bytes, (a.tt * a.n * 8 + 15) & ~15, a.n, op == kRotate ? 0 : (a.D + 3) & ~3,
                  op == kNormBwd ? (a.row_warps * a.D * 4 + 15) & ~15 : 0};
}

// A tile: tokens [token, token + count), heads [lo, lo + n) of either tensor.
struct Tile {
  uint32_t token;
  int count, lo[2], n[2], rows[2];
  DSLPG_DEV Tile(const HeadArgs& a, uint32_t tile) {
    if (a.parts == 1) {
      token = tile * a.tt;
      count = min(a.tt, static_cast<int>(a.tokens - token));
      lo[0] = lo[1] = 0;
      n[0] = a.heads[0];
      n[1] = a.heads[1];
    } else {
      token = tile / a.parts;
      count = 1;
      const int first = static_cast<int>(tile - token * a.parts) * a.part, last = first + a.part;
      lo[0] = min(first, a.heads[0]);
      n[0] = min(last, a.heads[0]) - lo[0];
      lo[1] = max(first - a.heads[0], 0);
      n[1] = min(max(last - a.heads[0], 0), a.heads[1]) - lo[1];
    }
    rows[0] = count * n[0];
    rows[1] = count * n[1];
  }
};

constexpr int kMaxTileTokens = 8;

// Where the k-th token of a CTA's tiles lies in a tensor with batch and sequence
// strides: divisions at the first tile only (at each with parts > 1).
struct Place {
  uint32_t s;
  int64_t at;
  DSLPG_DEV void seek(const HeadArgs& a, uint32_t token, int64_t batch, int64_t seq) {
    const uint32_t b = token / a.seq;
    s = token - b * a.seq;
    at = b * batch + s * seq;
  }
  DSLPG_DEV void next(const HeadArgs& a, int64_t step, int64_t carry) {
    s += a.s_step;
    at += step;
    if (s >= a.seq) {
      s -= a.seq;
      at += carry;
    }
  }
};
// Threads of a CTA at most. Whole 16-byte vectors need few warps, and more of them
// disturb one another's streams; narrower ones need the instruction slots. Measured
// (us) with 512, 640 and 768 threads: rotation of 29971 tokens of 16 + 16 heads of
// 128 in bf16 81.9, 83.9, 86.0, of 6845 of 16 + 16 of 72 in fp16 22.6, 20.6, 19.1;
// norm of 16384 tokens of 32 + 8 of 128 in bf16 65.7, 59.6, 59.5; its backward 90.0,
// 99.0, 119.
constexpr int tile_threads(int op, bool whole) {
  return op == kNorm ? 768 : (op == kRotate ? (whole ? 512 : 768) : (whole ? 512 : 640));
}
template <typename T, int V> constexpr bool kWholeVec = V == Elt<T>::kPerVec;

template <typename T, int V, bool INTER, int OP>
__global__ void __launch_bounds__(tile_threads(OP, kWholeVec<T, V>), 1)
    heads_tile_kernel(const __grid_constant__ HeadArgs a, unsigned long long limit_ns) {
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ volatile int abort_flag;
  constexpr int kBytes = Pack<T, V>::kBytes;
  constexpr bool NORM = OP != kRotate, BWD = OP == kNormBwd;
  const HeadSmem lay = head_smem(a, OP);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int vecs = a.D / V;
  uint64_t* freq = reinterpret_cast<uint64_t*>(smem + lay.freq());
  float* weights = reinterpret_cast<float*>(smem + lay.weight());
  const uint32_t stage0 = smem_u32(smem), full = smem_u32(smem + lay.bars()), empty = full + 8 * a.stages;
  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int s = 0; s < a.stages; ++s) {
      mbar_init(full + 8 * s, 1 + a.angle_warps);
      mbar_init(empty + 8 * s, a.groups);
    }
    fence_mbar_init();
  }
  for (int i = threadIdx.x; i < a.n; i += blockDim.x) freq[i] = turn_per_step(a.inv_freq[i]);
  if constexpr (NORM)
    for (int i = threadIdx.x; i < 2 * a.D; i += blockDim.x) {
      const int seg = i >= a.D, d = i - seg * a.D;
      weights[seg * lay.weight_floats + weight_slot<V>(d, vecs)] = load_any(a.w[seg], d, a.wdt);
    }
  __syncthreads();

  // Wait for a phase; false once any wait of this CTA ran out of time (the loops go on without waiting, so that all
  // of its warps end).
  auto wait = [&](uint32_t bar, uint32_t parity) {
    if (abort_flag) return false;
    if (mbar_wait(bar, parity, limit_ns)) return true;
    atomicAdd(&g_heads_timeouts, 1u);
    abort_flag = 1;
    return false;
  };

  if (warp == 0) {  // copies: lane 8 p + k has the k-th token of a tile in q, k, dq, dk (p)
    const int part = lane >> 3, k = lane & 7, seg = part & 1;
    const bool mine = part < (BWD ? 4 : 2) && k < a.tt && a.heads[seg] > 0;
    const bool is_dy = part >= 2;
    const T* base = static_cast<const T*>(is_dy ? a.dy[seg] : a.x[seg]);
    const int64_t st_b = is_dy ? a.dys[seg][0] : a.xs[seg][0], st_s = is_dy ? a.dys[seg][1] : a.xs[seg][1];
    const int64_t st_h = is_dy ? a.dys[seg][2] : a.xs[seg][2];
    const int64_t step = is_dy ? a.dy_step[seg] : a.x_step[seg], carry = is_dy ? a.dy_carry[seg] : a.x_carry[seg];
    const bool joined = st_h == a.D || a.heads[seg] == 1;  // heads that follow one another go in one copy
    const bool all_joined = __all_sync(0xffffffffu, joined || !mine);
    // Small tokens that follow one another too: one copy of them all, as the copy engine takes some 90 cycles for each
    // (99147 tokens of 4 + 1 heads of 64: 61.6 us against 75.9 with a copy a token). Larger ones are better apart (6845
    // tokens of 16 + 16 of 72 in fp16: 18.5 against 20.1).
    const int token_bytes = a.heads[seg] * a.row_bytes;
    const bool dense = all_joined && token_bytes <= 1024 && st_s == static_cast<int64_t>(a.heads[seg]) * a.D &&
                       (a.tokens <= a.seq || st_b == a.seq * st_s);
    Place place;
    uint32_t it = 0, st = 0, phase = 0;
    for (uint32_t tile = blockIdx.x; tile < a.tiles; tile += gridDim.x, ++it) {
      const Tile t(a, tile);
      if (it == 0 || a.parts > 1) place.seek(a, t.token + k, st_b, st_s);
      else place.next(a, step, carry);
      const int heads = seg ? t.n[1] : t.n[0];
      const T* src = base + place.at + (seg ? t.lo[1] : t.lo[0]) * st_h;
      const uint32_t bar = full + 8 * st;
      const uint32_t dst = stage0 + st * a.stage_bytes +
                           ((is_dy ? t.rows[0] + t.rows[1] : 0) + (seg ? t.rows[0] : 0) + k * heads) * a.row_bytes;
      const bool ok = mine && k < (dense ? 1 : t.count) && heads > 0;
      if (it >= static_cast<uint32_t>(a.stages) && !wait(empty + 8 * st, phase ^ 1u)) break;
      if (lane == 0) mbar_arrive_expect_tx(bar, (t.rows[0] + t.rows[1]) * a.row_bytes * (BWD ? 2 : 1));
      __syncwarp();
      auto copy = [&](uint32_t to, const T* from, int bytes) {
        asm volatile("cp.async.bulk.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(to),
                     "l"(from), "r"(bytes), "r"(bar)
                     : "memory");
      };
      if (all_joined) {
        if (ok) copy(dst, src, (dense ? t.count : 1) * heads * a.row_bytes);
      } else {
        for (int j = 0; j < (BWD ? 32 : 16); ++j) {  // a row a lane, token by token
          const int n = __shfl_sync(0xffffffffu, ok ? heads : 0, j);
          const int64_t sh = __shfl_sync(0xffffffffu, st_h, j);
          const uint32_t to = __shfl_sync(0xffffffffu, dst, j);
          const T* from = reinterpret_cast<const T*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(src), j));
          for (int h = lane; h < n; h += 32) copy(to + h * a.row_bytes, from + h * sh, a.row_bytes);
        }
      }
      if (++st == static_cast<uint32_t>(a.stages)) {
        st = 0;
        phase ^= 1u;
      }
    }
    // no copy is in flight when the CTA ends: the rows' warps wait for every full barrier, or (after a timeout) this does
    if (abort_flag)
      for (uint32_t s = 0; s < static_cast<uint32_t>(a.stages) && s < it; ++s)
        mbar_wait(full + 8 * s, s < st ? phase : phase ^ 1u, limit_ns / 8);
    return;
  }

  if (warp <= a.angle_warps) {  // angles, every angle_warps-th token of a tile
    uint32_t it = 0, st = 0, phase = 0;
    // this lane's position: axis lane & 3 of the tile's (lane >> 2)-th token of this warp
    const int mine = warp - 1 + (lane >> 2) * a.angle_warps, axis = lane & 3;
    Place place;
    auto position = [&](uint32_t tile, bool seek) {
      if (tile >= a.tiles) return 0ll;
      const Tile t(a, tile);
      if (seek || a.parts > 1) place.seek(a, t.token + mine, a.ps[1], a.ps[2]);
      else place.next(a, a.p_step, a.p_carry);
      if (mine >= t.count || axis >= a.axes) return 0ll;
      const int64_t j = place.at + axis * a.ps[0];
      return static_cast<long long>(a.pos64 ? static_cast<const int64_t*>(a.pos)[j] : static_cast<const int32_t*>(a.pos)[j]);
    };
    // loaded kAhead tiles before their use: a load from HBM takes longer than the angles of a tile
    constexpr int kAhead = 4;
    long long ahead[kAhead];
#pragma unroll
    for (int q = 0; q < kAhead; ++q) ahead[q] = position(blockIdx.x + q * gridDim.x, q == 0);
    bool more = true;
    for (uint32_t tile = blockIdx.x; more;) {
#pragma unroll
      for (int q = 0; q < kAhead; ++q) {
        if (tile >= a.tiles || (it >= static_cast<uint32_t>(a.stages) && !wait(empty + 8 * st, phase ^ 1u))) {
          more = false;
          break;
        }
        const int count = Tile(a, tile).count;
        float2* table = reinterpret_cast<float2*>(smem + lay.angles() + st * lay.angle_bytes);
        if (a.pairs) {
          for (int k = warp - 1, j = 0; k < count; k += 2 * a.angle_warps, j += 2) {
            const bool two = k + a.angle_warps < count;
#pragma unroll 1
            for (int i0 = 0; i0 < a.n; i0 += 32) {
              const int i = min(i0 + lane, a.n - 1), from = 4 * j + axis_of(a, i);
              const int64_t p0 = __shfl_sync(0xffffffffu, ahead[q], from), p1 = __shfl_sync(0xffffffffu, ahead[q], from + 4);
              const uint64_t f = freq[i];
              const float2 c0 = angle_of<sizeof(T) == 4>(p0, f, a.sign), c1 = angle_of<sizeof(T) == 4>(p1, f, a.sign);
              float2* to = table + k * a.n + angle_slot<V>(i, a.rot_units);
              *to = c0;  // (lanes past the last frequency write its value too)
              if (two) to[a.angle_warps * a.n] = c1;
            }
          }
        } else {
          for (int k = warp - 1, j = 0; k < count; k += a.angle_warps, ++j)
#pragma unroll 2
            for (int i0 = 0; i0 < a.n; i0 += 32) {
              const int i = i0 + lane;
              const int64_t at = __shfl_sync(0xffffffffu, ahead[q], 4 * j + axis_of(a, i));
              if (i < a.n)
                table[k * a.n + angle_slot<V>(i, a.rot_units)] = angle_of<sizeof(T) == 4>(at, freq[i], a.sign);
            }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(full + 8 * st);
        ahead[q] = position(tile + kAhead * gridDim.x, false);
        tile += gridDim.x;
        ++it;
        if (++st == static_cast<uint32_t>(a.stages)) {
          st = 0;
          phase ^= 1u;
        }
      }
    }
    return;
  }

  // rows
  const int me = warp - 1 - a.angle_warps;
  const Lane<INTER> ln(a, lane);
  const bool rotated = ln.active && ln.u < a.rot_units;
  const int b_off = (ln.ib - ln.ia) * V, b_bytes = b_off * static_cast<int>(sizeof(T));
  float da[V], db[V];  // norm backward: this lane's dw sums; a warp takes the rows of one tensor
  if constexpr (BWD) {
#pragma unroll
    for (int e = 0; e < V; ++e) da[e] = db[e] = 0.f;
  }
  const bool of_k = BWD && me >= a.q_warps;

  // Group g of the CTA's it-th tile: the groups of all its tiles go round the row warps (norm backward: q's and k's round
  // their own), and a warp waits for those tiles alone that hold one of its groups. A stage is free when all its groups
  // are done.
  uint32_t st = 0, phase = 0, tile = blockIdx.x;
  const int g_end = BWD && !of_k ? a.q_groups : a.groups, g_begin = of_k ? a.q_groups : 0;
  const int g_step = BWD ? (of_k ? a.row_warps - a.q_warps : a.q_warps) : a.row_warps;
  int g = of_k ? me - a.q_warps + a.q_groups : me;  // < g_end: no more warps than groups
  bool fresh = true;
  uint32_t base = 0;
  const float4* table = nullptr;
  T *out_q = nullptr, *out_k = nullptr;
  int rows_q = 0, rows_k = 0, q_groups = 0;
  while (tile < a.tiles) {
    if (fresh) {
      const Tile t(a, tile);
      wait(full + 8 * st, phase);
      base = stage0 + st * a.stage_bytes;
      table = reinterpret_cast<const float4*>(smem + lay.angles() + st * lay.angle_bytes);
      rows_q = t.rows[0];
      rows_k = t.rows[1];
      q_groups = BWD ? a.q_groups : (rows_q + a.rpw - 1) / a.rpw;
      out_q = static_cast<T*>(a.y[0]) + (static_cast<int64_t>(t.token) * a.heads[0] + t.lo[0]) * a.D + ln.ia * V;
      out_k = static_cast<T*>(a.y[1]) + (static_cast<int64_t>(t.token) * a.heads[1] + t.lo[1]) * a.D + ln.ia * V;
    }
    {
      const bool seg = BWD ? of_k : g >= q_groups;
      int r = (seg ? g - q_groups : g) * a.rpw + ln.sub;
      const bool ok = ln.active && r < (seg ? rows_k : rows_q);
      int row = r + (seg ? rows_q : 0);  // in the stage
      if (!ok) r = row = 0;
      const uint32_t src = base + row * a.row_bytes + ln.ia * kBytes;
      const uint32_t magic = seg ? a.magic[1] : a.magic[0];
      const int k = magic ? __umulhi(r, magic) : r;  // the row's token
      const float4* angles = table + k * (a.n / 2) + ln.u;
      const int dy_off = (rows_q + rows_k) * a.row_bytes;
      T* y = (seg ? out_k : out_q) + r * a.D;
      float xa[V], xb[V];
      lds_vec<T, V>(src, xa);
      lds_vec<T, V>(src + b_bytes, xb);
      if constexpr (!BWD) {
        if constexpr (NORM) {
          float sum[1] = {0.f}, sb = 0.f;
#pragma unroll
          for (int e = 0; e < V; ++e) {
            sum[0] += xa[e] * xa[e];
            sb += xb[e] * xb[e];
          }
          sum[0] += sb;
          row_sums(sum, a.units, ln.u, lane);
          const float rstd = rsqrtf(sum[0] * a.inv_d + a.eps);
          float w[V];
          const float* ws = weights + (seg ? lay.weight_floats : 0);
          read_weights<V>(ws, ln.ia, vecs, w);
#pragma unroll
          for (int e = 0; e < V; ++e) xa[e] *= rstd * w[e];
          read_weights<V>(ws, ln.ib, vecs, w);
#pragma unroll
          for (int e = 0; e < V; ++e) xb[e] *= rstd * w[e];
        }
        if (rotated) turn<V, INTER>(xa, xb, angles, a.rot_units);
        if (ok) {
          st_vec<T, V>(y, xa);
          st_vec<T, V>(y + b_off, xb);
        }
      } else {
        float ga[V], gb[V], wa[V], wb[V];
        lds_vec<T, V>(src + dy_off, ga);
        lds_vec<T, V>(src + dy_off + b_bytes, gb);
        if (rotated) turn<V, INTER>(ga, gb, angles, a.rot_units);
        const float* ws = weights + (seg ? lay.weight_floats : 0);
        read_weights<V>(ws, ln.ia, vecs, wa);
        read_weights<V>(ws, ln.ib, vecs, wb);
        float sum[2] = {0.f, 0.f}, sb = 0.f, cb = 0.f;
#pragma unroll
        for (int e = 0; e < V; ++e) {
          sum[0] += xa[e] * xa[e];
          sb += xb[e] * xb[e];
          wa[e] *= ga[e];
          wb[e] *= gb[e];
          sum[1] += wa[e] * xa[e];
          cb += wb[e] * xb[e];
        }
        sum[0] += sb;
        sum[1] += cb;
        row_sums(sum, a.units, ln.u, lane);
        if (ok) {
          const float rstd = rsqrtf(sum[0] * a.inv_d + a.eps), c = rstd * rstd * (sum[1] * a.inv_d);
#pragma unroll
          for (int e = 0; e < V; ++e) {
            da[e] += ga[e] * (xa[e] * rstd);
            db[e] += gb[e] * (xb[e] * rstd);
            wa[e] = rstd * (wa[e] - xa[e] * c);
            wb[e] = rstd * (wb[e] - xb[e] * c);
          }
          st_vec<T, V>(y, wa);
          st_vec<T, V>(y + b_off, wb);
        }
      }
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(empty + 8 * st);
    g += g_step;
    fresh = g >= g_end;
    while (g >= g_end) {
      g -= g_end - g_begin;
      tile += gridDim.x;
      if (++st == static_cast<uint32_t>(a.stages)) {
        st = 0;
        phase ^= 1u;
      }
    }
  }

  if constexpr (BWD) {
    // dw: the rows of a group, then the tensor's warps, then (heads_dw_kernel) the CTAs, each in a fixed order, so that
    // the same call gives the same bits
    float* sums = reinterpret_cast<float*>(smem + lay.sums());  // [row warps][D]
#pragma unroll
    for (int e = 0; e < V; ++e) {
      float ta = da[e], tb = db[e];
      for (int r = 1; r < a.rpw; ++r) {
        ta += __shfl_sync(0xffffffffu, da[e], (ln.u + r * a.units) & 31);
        tb += __shfl_sync(0xffffffffu, db[e], (ln.u + r * a.units) & 31);
      }
      if (ln.active && ln.sub == 0) {
        sums[me * a.D + ln.ia * V + e] = ta;
        sums[me * a.D + ln.ib * V + e] = tb;
      }
    }
    asm volatile("bar.sync 1, %0;" ::"r"(a.row_warps * 32) : "memory");
    for (int i = me * 32 + lane; i < 2 * a.D; i += a.row_warps * 32) {
      const int seg = i >= a.D, d = i - seg * a.D;
      float t = 0.f;
      for (int k = seg ? a.q_warps : 0; k < (seg ? a.row_warps : a.q_warps); ++k) t += sums[k * a.D + d];
      a.partial[static_cast<int64_t>(blockIdx.x) * 2 * a.D + i] = t;
    }
  }
}

// A token and one of its groups.
struct Cursor {
  uint32_t b, s;
  int g;
  DSLPG_DEV Cursor(const HeadArgs& a, int64_t at, int all) {
    const uint32_t token = static_cast<uint32_t>(at / all);
    g = static_cast<int>(at - static_cast<int64_t>(token) * all);
    b = token / a.seq;
    s = token - b * a.seq;
  }
  DSLPG_DEV bool next(const HeadArgs& a, int all) {  // whether a new token begins
    if (++g < all) return false;
    g = 0;
    if (++s == a.seq) {
      s = 0;
      ++b;
    }
    return true;
  }
};

// dw[seg][d] = the sum of the CTAs' partial rows: 8 threads a column, each every 8th row, merged in order.
__global__ void __launch_bounds__(256) heads_dw_kernel(const float* partial, int ctas, int D, float* dq, float* dk) {
  __shared__ float part[8][32];
  wait_for_primary();
  const int col = threadIdx.x & 31, row = threadIdx.x >> 5;
  const int d = blockIdx.x * 32 + col, seg = blockIdx.y;
  float t = 0.f;
  if (d < D)
    for (int r = row; r < ctas; r += 8) t += partial[(static_cast<int64_t>(r) * 2 + seg) * D + d];
  part[row][col] = t;
  __syncthreads();
  if (row == 0 && d < D) {
#pragma unroll
    for (int k = 1; k < 8; ++k) t += part[k][col];
    (seg ? dk : dq)[d] = t;
  }
}

// Any head size, alignment and stride: a warp takes one row at a time with
// scalar accesses, reading it twice (the second time from L1 / L2). `dw` sums
// are kept per warp in shared memory.
template <typename T, bool NORM, bool BWD>
__global__ void __launch_bounds__(128) heads_any_kernel(const __grid_constant__ HeadArgs a) {
  extern __shared__ __align__(128) unsigned char smem[];
  const int wstride = (a.D + 3) & ~3;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  uint64_t* freq = reinterpret_cast<uint64_t*>(smem);                     // [n]
  float2* cs = reinterpret_cast<float2*>(freq + a.n) + warp * a.n;    // [warps][n]
  float* all_sums = reinterpret_cast<float*>(smem + 8 * a.n * (warps + 1));
  float* sums = all_sums + warp * 2 * wstride;                        // BWD: [warps][2][D]
  for (int i = threadIdx.x; i < a.n; i += blockDim.x) freq[i] = turn_per_step(a.inv_freq[i]);
  __syncthreads();
  const int all = a.heads[0] + a.heads[1];
  const int64_t total = static_cast<int64_t>(a.tokens) * all, mine = static_cast<int64_t>(blockIdx.x) * warps + warp;
  const int64_t share = static_cast<int64_t>(gridDim.x) * warps;
  const int64_t lo_row = total * mine / share, hi_row = total * (mine + 1) / share;
  if constexpr (BWD)
    for (int d = lane; d < 2 * wstride; d += 32) sums[d] = 0.f;
  const int n = a.n, D = a.D;
  // Index of the two members of pair i.
  auto lo = [&](int i) { return a.interleaved ? 2 * i : i; };
  auto hi = [&](int i) { return a.interleaved ? 2 * i + 1 : i + n; };
  if (hi_row > lo_row) {
    Cursor at(a, lo_row, all);
    bool fresh = true;
    for (int64_t row = lo_row; row < hi_row; ++row, fresh = at.next(a, all)) {
      const uint32_t b = at.b, s = at.s;
      if (fresh) {
        fill_angles<sizeof(T) == 4>(a, freq, cs, lane_position(a, b * a.ps[1] + s * a.ps[2], lane), lane);
      }
      const int seg = at.g >= a.heads[0], head = at.g - (seg ? a.heads[0] : 0);
      const T* src = static_cast<const T*>(a.x[seg]) + b * a.xs[seg][0] + s * a.xs[seg][1] + head * a.xs[seg][2];
      T* dst = static_cast<T*>(a.y[seg]) + ((static_cast<int64_t>(b) * a.seq + s) * a.heads[seg] + head) * D;
      float rstd = 1.f;
      if constexpr (NORM) {
        float ss = 0.f;
        for (int d = lane; d < D; d += 32) {
          const float v = to_f(src[d]);
          ss += v * v;
        }
        rstd = rsqrtf(warp_reduce<SumOp>(ss) * a.inv_d + a.eps);
      }
      if constexpr (!BWD) {
        auto u = [&](int d) { return NORM ? to_f(src[d]) * rstd * load_any(a.w[seg], d, a.wdt) : to_f(src[d]); };
        for (int i = lane; i < n; i += 32) {
          const float x0 = u(lo(i)), x1 = u(hi(i));
          dst[lo(i)] = from_f<T>(x0 * cs[i].x - x1 * cs[i].y);
          dst[hi(i)] = from_f<T>(x1 * cs[i].x + x0 * cs[i].y);
        }
        for (int d = 2 * n + lane; d < D; d += 32) dst[d] = from_f<T>(u(d));
      } else {
        const T* dy = static_cast<const T*>(a.dy[seg]) + b * a.dys[seg][0] + s * a.dys[seg][1] + head * a.dys[seg][2];
        auto w = [&](int d) { return load_any(a.w[seg], d, a.wdt); };
        auto pair = [&](int i, float& g0, float& g1) {
          const float y0 = to_f(dy[lo(i)]), y1 = to_f(dy[hi(i)]);
          g0 = y0 * cs[i].x - y1 * cs[i].y;
          g1 = y1 * cs[i].x + y0 * cs[i].y;
        };
        float cc = 0.f;
        for (int i = lane; i < n; i += 32) {
          float g0, g1;
          pair(i, g0, g1);
          cc += w(lo(i)) * g0 * to_f(src[lo(i)]) + w(hi(i)) * g1 * to_f(src[hi(i)]);
        }
        for (int d = 2 * n + lane; d < D; d += 32) cc += w(d) * to_f(dy[d]) * to_f(src[d]);
        const float k = rstd * rstd * (warp_reduce<SumOp>(cc) * a.inv_d);
        auto put = [&](int d, float g) {
          const float v = to_f(src[d]);
          sums[seg * wstride + d] += g * (v * rstd);  // feature d is the same lane's in every row
          dst[d] = from_f<T>(rstd * (w(d) * g - v * k));
        };
        for (int i = lane; i < n; i += 32) {
          float g0, g1;
          pair(i, g0, g1);
          put(lo(i), g0);
          put(hi(i), g1);
        }
        for (int d = 2 * n + lane; d < D; d += 32) put(d, to_f(dy[d]));
      }
    }
  }
  if constexpr (BWD) {
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * D; i += blockDim.x) {
      const int seg = i >= D, d = i - seg * D;
      float t = 0.f;
      for (int k = 0; k < warps; ++k) t += all_sums[(2 * k + seg) * wstride + d];
      a.partial[static_cast<int64_t>(blockIdx.x) * 2 * D + i] = t;
    }
  }
}

namespace {

constexpr int kMaxHeadDim = 1024;
constexpr int kPartialRows = 1184;  // CTAs of a norm backward at most (8 for each of 148 SMs), each with a row for q and one for k

constexpr int kTileSmem = 216 * 1024;  // of the 227 KB that a CTA may have
constexpr int kAnyBlock = 128;

uint32_t magic_of(int heads) { return heads > 1 ? static_cast<uint32_t>(((1ull << 32) + heads - 1) / heads) : 0; }

// Cut the work into tiles. A tile holds up to 8 tokens and 80 KB (rotation alone:
// 40 KB), fewer tokens while that leaves SMs without four tiles each, and less
// than a token where one token is too large or there are not tokens enough.
// Measured (us) with 20, 40 and 80 KB: norm forward of 16384 tokens of 32 + 8
// heads of 128 in bf16 90.2, 61.6, 59.5; rotation of 29971 tokens of 16 + 16 heads
// 135, 86.0, 90.8 (with 768 threads).
template <typename T> void set_tiles(HeadArgs& a, int op) {
  const int heads = a.heads[0] + a.heads[1], copies = op == kNormBwd ? 2 : 1, sms = sm_count();
  a.row_bytes = a.D * static_cast<int>(sizeof(T));
  const int64_t row = static_cast<int64_t>(a.row_bytes) * copies, token = row * heads;
  const int64_t want = (op == kRotate ? 40 : 80) * 1024;
  a.parts = 1;
  a.part = heads;
  a.tt = 1;
  while (a.tt < kMaxTileTokens && token * a.tt * 2 <= want && static_cast<int64_t>(a.tokens) >= 4ll * a.tt * sms) a.tt *= 2;
  if (a.tt == 1) {
    // at most 32 KB of rows, and as many parts as leave every SM one, but whole groups of rows
    int64_t part = heads;
    if (token > 32 * 1024) part = 32 * 1024 / row;
    const int64_t spare = (sms + static_cast<int64_t>(a.tokens) - 1) / a.tokens;
    if (heads / spare < part) part = heads / spare;
    part = part < 1 ? a.rpw : (part + a.rpw - 1) / a.rpw * a.rpw;
    if (part < heads) {
      a.part = static_cast<int>(part);
      a.parts = (heads + a.part - 1) / a.part;
    }
  }
  a.tiles = a.parts == 1 ? (a.tokens + a.tt - 1) / a.tt : a.tokens * a.parts;
  a.stage_bytes = static_cast<int>((row * (a.parts == 1 ? static_cast<int64_t>(heads) * a.tt : a.part) + 127) & ~127ll);
  a.magic[0] = a.parts == 1 ? magic_of(a.heads[0]) : magic_of(1 << 30);
  a.magic[1] = a.parts == 1 ? magic_of(a.heads[1]) : magic_of(1 << 30);
}

template <typename T, int V, bool INTER, int OP>
cudaError_t launch_tile(HeadArgs a, float* dwq, float* dwk, cudaStream_t st) {
  a.rot_units = a.n / V;
  a.units = a.D / (2 * V);
  a.rpw = 32 / a.units;
  set_tiles<T>(a, OP);
  const int heads = a.heads[0] + a.heads[1];
  const int part_groups = (a.part + a.rpw - 1) / a.rpw;
  a.q_groups = a.parts == 1 ? (a.heads[0] * a.tt + a.rpw - 1) / a.rpw : part_groups;
  const int k_groups = a.parts == 1 ? (a.heads[1] * a.tt + a.rpw - 1) / a.rpw : (OP == kNormBwd ? part_groups : 1);
  a.groups = a.q_groups + k_groups;
  // Warps: one for copies; some for angles; the rest for rows, no more than a tile has groups. One angle warp for two
  // tokens (backward, whose rows take twice the time: for four).
  a.angle_warps = OP == kNormBwd ? (a.tt + 3) / 4 : (a.tt + 1) / 2;
  // An angle is a chain of a few hundred cycles, so two tokens' run side by side, but not in a rotation whose rows weigh
  // more (16 whole heads of 16-bit elements a token): there the slower angles keep the loads and stores of all SMs in a
  // better order; why was not found. Single / pairs, in us, for 45000 tokens in bf16 of 6 + 6 heads of 128: 57.7 / 51.3,
  // of 8 + 4 of 256: 140 / 103, of 8 + 8 of 128: 63.7 / 71.2, of 16 + 16: 121 / 143; 99147 in float32 of 8 + 8 of 128:
  // 265 / 295.
  a.pairs = OP != kRotate || static_cast<int64_t>(heads) * a.row_bytes < 64ll * a.n;
  a.row_warps = tile_threads(OP, kWholeVec<T, V>) / 32 - 1 - a.angle_warps;
  if (a.row_warps > a.groups) {  // (4 + 1 heads of 96, 99147 tokens: norm 113 us without the spare warps, 90 with them)
    a.angle_warps = std::min(a.tt, a.angle_warps + a.row_warps - a.groups);
    a.row_warps = a.groups;
  }
  // The q : k split of the row warps that ends first: the largest share of groups a warp, as fractions over the other's
  // warps. Exchanging the sums of two tensors in one warp took 50 instructions a time instead.
  a.q_warps = k_groups ? (a.q_groups ? 1 : 0) : a.row_warps;
  auto longer = [&](int q) {
    const int k = a.row_warps - q;
    return std::max(q ? a.q_groups * 1.0 / q : (a.q_groups ? 1e9 : 0.0), k ? k_groups * 1.0 / k : (k_groups ? 1e9 : 0.0));
  };
  for (int q = a.q_warps + 1; q <= a.row_warps; ++q)
    if (longer(q) < longer(a.q_warps)) a.q_warps = q;
  const int block = 32 * (1 + a.angle_warps + a.row_warps);
  const void* fn = reinterpret_cast<const void*>(&heads_tile_kernel<T, V, INTER, OP>);
  const int grid = static_cast<int>(a.tiles < static_cast<uint32_t>(sm_count()) ? a.tiles : sm_count());
  const int mine = static_cast<int>((a.tiles + grid - 1) / grid);  // tiles of a CTA at most
  for (a.stages = mine < 16 ? mine : 16; a.stages > 1 && head_smem(a, OP).total() > kTileSmem; --a.stages) {
  }
  const int64_t ahead = static_cast<int64_t>(grid) * a.tt, db = ahead / a.seq, ds = ahead % a.seq;
  for (int seg = 0; seg < 2; ++seg) {
    a.x_step[seg] = db * a.xs[seg][0] + ds * a.xs[seg][1];
    a.x_carry[seg] = a.xs[seg][0] - static_cast<int64_t>(a.seq) * a.xs[seg][1];
    a.dy_step[seg] = db * a.dys[seg][0] + ds * a.dys[seg][1];
    a.dy_carry[seg] = a.dys[seg][0] - static_cast<int64_t>(a.seq) * a.dys[seg][1];
  }
  a.p_step = db * a.ps[1] + ds * a.ps[2];
  a.p_carry = a.ps[1] - static_cast<int64_t>(a.seq) * a.ps[2];
  a.s_step = static_cast<uint32_t>(ds);
  const size_t smem = head_smem(a, OP).total();
  if (cudaError_t e = allow_dynamic_smem(fn, smem)) return e;
  heads_tile_kernel<T, V, INTER, OP><<<grid, block, smem, st>>>(a, kWaitLimitNs);
  if (cudaError_t e = cudaGetLastError()) return e;
  if constexpr (OP == kNormBwd) return launch_dependent(heads_dw_kernel, dim3((a.D + 31) / 32, 2), 256, st, static_cast<const float*>(a.partial), grid, a.D, dwq, dwk);
  return cudaSuccess;
}

template <typename T, bool NORM, bool BWD>
cudaError_t launch_any(HeadArgs a, float* dwq, float* dwk, cudaStream_t st) {
  const size_t smem = (BWD ? static_cast<size_t>((a.D + 3) & ~3) * 8 * (kAnyBlock / 32) : 0) +
                      static_cast<size_t>(kAnyBlock / 32 + 1) * a.n * 8;
  const void* fn = reinterpret_cast<const void*>(&heads_any_kernel<T, NORM, BWD>);
  if (cudaError_t e = allow_dynamic_smem(fn, smem)) return e;
  const int64_t rows = static_cast<int64_t>(a.tokens) * (a.heads[0] + a.heads[1]);
  int grid = persistent_grid(fn, kAnyBlock, smem, (rows + kAnyBlock / 32 - 1) / (kAnyBlock / 32));
  if (BWD && grid > kPartialRows) grid = kPartialRows;
  heads_any_kernel<T, NORM, BWD><<<grid, kAnyBlock, smem, st>>>(a);
  if (cudaError_t e = cudaGetLastError()) return e;
  if constexpr (BWD) return launch_dependent(heads_dw_kernel, dim3((a.D + 31) / 32, 2), 256, st, static_cast<const float*>(a.partial), grid, a.D, dwq, dwk);
  return cudaSuccess;
}

// Whether rows can be cut into units of two V-element vectors.
template <typename T>
bool fits(const HeadArgs& a, int V) {
  // n % V: half of the rotated features, or 2 V of them interleaved; the others in pairs of vectors too
  return a.D % (2 * V) == 0 && a.n % V == 0 && a.D / (2 * V) <= 32;
}

// Whether rows can be copied in bulk: 16-byte addresses and sizes.
template <typename T>
bool copies_fit(const HeadArgs& a, bool bwd) {
  constexpr int E = Elt<T>::kPerVec;
  if (a.D % E) return false;
  for (int seg = 0; seg < 2; ++seg) {
    if (!aligned(a.x[seg], 16) || !aligned(a.y[seg], 16) || (bwd && !aligned(a.dy[seg], 16))) return false;
    for (int k = 0; k < 3; ++k)
      if (a.xs[seg][k] % E || (bwd && a.dys[seg][k] % E)) return false;
  }
  return true;
}

template <typename T, int V, bool INTER>
cudaError_t launch_v(const HeadArgs& a, bool norm, bool bwd, float* dwq, float* dwk, cudaStream_t st) {
  if (bwd) return launch_tile<T, V, INTER, kNormBwd>(a, dwq, dwk, st);
  return norm ? launch_tile<T, V, INTER, kNorm>(a, dwq, dwk, st) : launch_tile<T, V, INTER, kRotate>(a, dwq, dwk, st);
}

template <typename T>
cudaError_t dispatch(HeadArgs a, bool norm, bool bwd, float* dwq, float* dwk, cudaStream_t st) {
  constexpr int E = Elt<T>::kPerVec;
  if (kernel_path() != DSLPG_PATH_STREAM && copies_fit<T>(a, bwd)) {
    if (fits<T>(a, E))
      return a.interleaved ? launch_v<T, E, true>(a, norm, bwd, dwq, dwk, st)
                           : launch_v<T, E, false>(a, norm, bwd, dwq, dwk, st);
    if (fits<T>(a, E / 2))
      return a.interleaved ? launch_v<T, E / 2, true>(a, norm, bwd, dwq, dwk, st)
                           : launch_v<T, E / 2, false>(a, norm, bwd, dwq, dwk, st);
    if constexpr (E > 4)
      if (fits<T>(a, 2))  // pairs in fours but not in eights (36 of 72 features)
        return a.interleaved ? launch_v<T, 2, true>(a, norm, bwd, dwq, dwk, st)
                             : launch_v<T, 2, false>(a, norm, bwd, dwq, dwk, st);
  }
  if (bwd) return launch_any<T, true, true>(a, dwq, dwk, st);
  return norm ? launch_any<T, true, false>(a, dwq, dwk, st) : launch_any<T, false, false>(a, dwq, dwk, st);
}

cudaError_t dispatch_dtype(const HeadArgs& a, int dt, bool norm, bool bwd, float* dwq, float* dwk, cudaStream_t st) {
  switch (dt) {
    case DSLPG_F32: return dispatch<float>(a, norm, bwd, dwq, dwk, st);
    case DSLPG_F16: return dispatch<__half>(a, norm, bwd, dwq, dwk, st);
    default: return dispatch<__nv_bfloat16>(a, norm, bwd, dwq, dwk, st);
  }
}

// Checks what every entry point takes and fills the shared arguments.
int common_args(HeadArgs& a, const dslpg_heads* h, const void* positions, const float* inv_freq, float sign) {
  if (h == nullptr || positions == nullptr || inv_freq == nullptr) return DSLPG_ERR_NULL_POINTER;
  if (!is_float_dtype(h->dtype) || (h->positions_dtype != DSLPG_I32 && h->positions_dtype != DSLPG_I64))
    return DSLPG_ERR_BAD_DTYPE;
  constexpr int64_t kMost = 1ll << 30;
  if (h->batch < 0 || h->seq < 0 || h->q_heads < 0 || h->k_heads < 0 || h->q_heads > kMost || h->k_heads > kMost ||
      h->head_dim < 1 || h->head_dim > kMaxHeadDim || h->rotary_dim < 2 || h->rotary_dim > h->head_dim ||
      h->rotary_dim % 2)
    return DSLPG_ERR_BAD_SHAPE;
  // items of a launch (tokens times heads) are counted in 32 bits, with room for one more grid step
  const int64_t heads = h->q_heads + h->k_heads;
  if (h->batch > 0 && h->seq > 0 && heads > 0 && (h->batch > kMost / h->seq || h->batch * h->seq > kMost / heads))
    return DSLPG_ERR_BAD_SHAPE;
  if (h->axes < 1 || h->axes > 4) return DSLPG_ERR_BAD_ARGUMENT;
  int64_t sum = 0;
  for (int k = 0; k < h->axes; ++k) {
    if (h->sections[k] < 0 || h->sections[k] > h->rotary_dim) return DSLPG_ERR_BAD_ARGUMENT;
    sum += h->sections[k];
    if (k < 3) a.bound[k] = static_cast<int>(sum);
  }
  if (sum != h->rotary_dim / 2) return DSLPG_ERR_BAD_ARGUMENT;
  for (int k = h->axes - 1; k < 3; ++k) a.bound[k] = static_cast<int>(h->rotary_dim / 2);
  a.pos = positions;
  a.inv_freq = inv_freq;
  a.tokens = static_cast<uint32_t>(h->batch * h->seq);
  a.seq = static_cast<uint32_t>(h->seq);
  a.heads[0] = static_cast<int>(h->q_heads);
  a.heads[1] = static_cast<int>(h->k_heads);
  a.D = static_cast<int>(h->head_dim);
  a.n = static_cast<int>(h->rotary_dim / 2);
  // the stride of an extent of one is never used, whatever it says
  const int64_t extents[2][3] = {{h->batch, h->seq, h->q_heads}, {h->batch, h->seq, h->k_heads}};
  const int64_t pos_extents[3] = {h->axes, h->batch, h->seq};
  for (int k = 0; k < 3; ++k) {
    a.xs[0][k] = extents[0][k] > 1 ? h->q_strides[k] : 0;
    a.xs[1][k] = extents[1][k] > 1 ? h->k_strides[k] : 0;
    a.dys[0][k] = extents[0][k] > 1 ? h->dq_strides[k] : 0;
    a.dys[1][k] = extents[1][k] > 1 ? h->dk_strides[k] : 0;
    a.ps[k] = pos_extents[k] > 1 ? h->position_strides[k] : 0;
  }
  a.axes = h->axes;
  a.pos64 = h->positions_dtype == DSLPG_I64 ? 1 : 0;
  a.interleaved = h->interleaved ? 1 : 0;
  a.inv_d = 1.0f / static_cast<float>(a.D);
  a.sign = sign;
  return DSLPG_OK;
}

// q's or k's pointers may be null when it has no heads.
bool missing(const HeadArgs& a, bool bwd) {
  for (int seg = 0; seg < 2; ++seg)
    if (a.heads[seg] > 0 && (!a.x[seg] || !a.y[seg] || (bwd && !a.dy[seg]))) return true;
  return false;
}

bool eps_ok(float eps) { return eps >= 0.f && eps < kPosInf; }

int run_rope(const void* q, const void* k, const void* positions, const float* inv_freq, void* q_out, void* k_out,
             const dslpg_heads* h, float sign, cudaStream_t stream) {
  HeadArgs a{};
  if (int rc = common_args(a, h, positions, inv_freq, sign)) return rc;
  if (a.tokens == 0 || a.heads[0] + a.heads[1] == 0) return DSLPG_OK;
  a.x[0] = q;
  a.x[1] = k;
  a.y[0] = q_out;
  a.y[1] = k_out;
  if (missing(a, false)) return DSLPG_ERR_NULL_POINTER;
  return static_cast<int>(dispatch_dtype(a, h->dtype, false, false, nullptr, nullptr, stream));
}

}  // namespace

unsigned int take_wait_timeouts_heads() {
  unsigned int v = 0, zero = 0;
  cudaMemcpyFromSymbol(&v, g_heads_timeouts, sizeof(v));
  cudaMemcpyToSymbol(g_heads_timeouts, &zero, sizeof(zero));
  return v;
}

}  // namespace dslpg

using namespace dslpg;

extern "C" int dslpg_rope_fwd(const void* q, const void* k, const void* positions, const float* inv_freq, void* q_out,
                              void* k_out, const dslpg_heads* h, cudaStream_t stream) {
  return run_rope(q, k, positions, inv_freq, q_out, k_out, h, 1.f, stream);
}

extern "C" int dslpg_rope_bwd(const void* dq_out, const void* dk_out, const void* positions, const float* inv_freq,
                              void* dq, void* dk, const dslpg_heads* h, cudaStream_t stream) {
  return run_rope(dq_out, dk_out, positions, inv_freq, dq, dk, h, -1.f, stream);
}

extern "C" int dslpg_qk_norm_rope_fwd(const void* q, const void* k, const void* q_weight, const void* k_weight,
                                      const void* positions, const float* inv_freq, void* q_out, void* k_out,
                                      const dslpg_heads* h, float eps, cudaStream_t stream) {
  if (!q_weight || !k_weight) return DSLPG_ERR_NULL_POINTER;
  HeadArgs a{};
  if (int rc = common_args(a, h, positions, inv_freq, 1.f)) return rc;
  if (!is_float_dtype(h->weight_dtype)) return DSLPG_ERR_BAD_DTYPE;
  if (!eps_ok(eps)) return DSLPG_ERR_BAD_EPS;
  if (a.tokens == 0 || a.heads[0] + a.heads[1] == 0) return DSLPG_OK;
  a.x[0] = q;
  a.x[1] = k;
  a.w[0] = q_weight;
  a.w[1] = k_weight;
  a.wdt = h->weight_dtype;
  a.y[0] = q_out;
  a.y[1] = k_out;
  a.eps = eps;
  if (missing(a, false)) return DSLPG_ERR_NULL_POINTER;
  return static_cast<int>(dispatch_dtype(a, h->dtype, true, false, nullptr, nullptr, stream));
}

extern "C" int dslpg_qk_norm_rope_bwd_workspace_bytes(int64_t head_dim, int64_t* bytes) {
  if (!bytes) return DSLPG_ERR_NULL_POINTER;
  if (head_dim < 1 || head_dim > kMaxHeadDim) return DSLPG_ERR_BAD_SHAPE;
  *bytes = kPartialRows * 2 * head_dim * 4;
  return DSLPG_OK;
}

extern "C" int dslpg_qk_norm_rope_bwd(const void* dq_out, const void* dk_out, const void* q, const void* k,
                                      const void* q_weight, const void* k_weight, const void* positions,
                                      const float* inv_freq, void* dq, void* dk, float* dq_weight, float* dk_weight,
                                      const dslpg_heads* h, float eps, void* workspace, int64_t workspace_bytes,
                                      cudaStream_t stream) {
  if (!q_weight || !k_weight || !dq_weight || !dk_weight || !workspace) return DSLPG_ERR_NULL_POINTER;
  HeadArgs a{};
  if (int rc = common_args(a, h, positions, inv_freq, -1.f)) return rc;
  if (!is_float_dtype(h->weight_dtype)) return DSLPG_ERR_BAD_DTYPE;
  if (!eps_ok(eps)) return DSLPG_ERR_BAD_EPS;
  if (workspace_bytes < static_cast<int64_t>(kPartialRows) * 2 * a.D * 4 || !aligned(workspace, 16)) return DSLPG_ERR_BAD_ARGUMENT;
  if (a.tokens == 0 || a.heads[0] + a.heads[1] == 0) {
    cudaError_t e = cudaMemsetAsync(dq_weight, 0, static_cast<size_t>(a.D) * 4, stream);
    if (e == cudaSuccess) e = cudaMemsetAsync(dk_weight, 0, static_cast<size_t>(a.D) * 4, stream);
    return static_cast<int>(e);
  }
  a.x[0] = q;
  a.x[1] = k;
  a.dy[0] = dq_out;
  a.dy[1] = dk_out;
  a.w[0] = q_weight;
  a.w[1] = k_weight;
  a.wdt = h->weight_dtype;
  a.y[0] = dq;
  a.y[1] = dk;
  a.eps = eps;
  a.partial = static_cast<float*>(workspace);
  if (missing(a, true)) return DSLPG_ERR_NULL_POINTER;
  return static_cast<int>(dispatch_dtype(a, h->dtype, true, true, dq_weight, dk_weight, stream));
}
