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
// Angles: pos * f_i is formed in 64 bits as turns, pos * (f_i / 2 pi), its
// whole turns are dropped exactly, and the fraction goes to sincospi in 32
// bits; far positions (1e6 and more) keep the cosine to 32-bit accuracy. The
// n angles of a token serve all of its heads, so one warp takes a token (or
// part of its heads when there are few tokens), computes the angles once into
// its own slice of shared memory and then walks the heads.
//
// Lanes: a row is cut into units of two V-element vectors that hold both
// members of V rotated pairs (vectors u and u + n/V; interleaved 2u and
// 2u + 1), so the rotation needs no exchange between lanes; the features
// past R are units of two neighbouring vectors. L lanes (a power of two) hold
// a row, 32 / L rows go through a warp at a time.
#include "common.cuh"
#include "pipe.cuh"

namespace dslpg {

struct HeadArgs {
  const void* x[2];    // q, k: the rows (rotation backward: dy)
  const void* dy[2];   // norm backward: the gradients of the outputs
  void* y[2];          // outputs, dense [tokens, heads, D]
  const void* w[2];    // [D] weights
  const void* pos;
  const float* inv_freq;
  float* partial;      // norm backward: [CTAs][D] sums for dw
  int64_t xs[2][3];    // batch, sequence and head strides of x
  int64_t dys[2][3];
  int64_t ps[3];       // axis, batch and sequence strides of pos
  uint32_t tokens, seq;
  int heads[2];
  int D, n;            // features; rotated pairs
  int bound[3];        // first frequency of axes 1, 2, 3
  int rot_units, units, log_l;
  int groups[2];       // groups of 32 / L heads
  uint32_t chunk, chunks;  // groups per item, items per token (norm backward: of q's CTAs)
  uint32_t chunk_k, chunks_k;  // norm backward: of k's CTAs
  int q_ctas;          // norm backward: the first q_ctas CTAs take q, the others k
  int wdt, pos64, interleaved;
  float eps, inv_d, sign;
};

// V elements of T in 32-bit words.
template <typename T, int V> struct Pack {
  static constexpr int kWords = V * static_cast<int>(sizeof(T)) / 4;
  uint32_t w[kWords];
};

template <typename T, int V> DSLPG_DEV void ld_pack(Pack<T, V>& p, const T* src) {
  if constexpr (Pack<T, V>::kWords == 4) {
    const Vec16 v = ld_stream(src);
#pragma unroll
    for (int i = 0; i < 4; ++i) p.w[i] = v.w[i];
  } else {
    static_assert(Pack<T, V>::kWords == 2, "8- or 16-byte vectors");
    asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(p.w[0]), "=r"(p.w[1]) : "l"(src));
  }
}

template <typename T, int V> DSLPG_DEV void st_pack(T* dst, const float (&f)[V]) {
  uint32_t w[Pack<T, V>::kWords];
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < V; ++i) w[i] = __float_as_uint(f[i]);
  } else {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) w[i] = pack2<T>(f[2 * i], f[2 * i + 1]);
  }
  if constexpr (Pack<T, V>::kWords == 4) st_stream(dst, Vec16{{w[0], w[1], w[2], w[3]}});
  else st_stream8(dst, w[0], w[1]);
}

template <typename T, int V> DSLPG_DEV void unpack_to(const Pack<T, V>& p, float (&f)[V]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = __uint_as_float(p.w[i]);
  } else {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) upk2(unpack_pair<T>(Vec16{{p.w[i], 0u, 0u, 0u}}, 0), f[2 * i], f[2 * i + 1]);
  }
}

// Cosines and sines of token (b, s) for this warp: cs[i] = (cos, sin) of frequency i.
DSLPG_DEV void fill_angles(const HeadArgs& a, float2* cs, uint32_t b, uint32_t s, int lane) {
  const int64_t at = b * a.ps[1] + s * a.ps[2];
  for (int i = lane; i < a.n; i += 32) {
    const int axis = (i >= a.bound[0]) + (i >= a.bound[1]) + (i >= a.bound[2]);
    const int64_t j = at + axis * a.ps[0];
    const double p = a.pos64 ? static_cast<double>(static_cast<const int64_t*>(a.pos)[j])
                             : static_cast<double>(static_cast<const int32_t*>(a.pos)[j]);
    const double turns = p * (static_cast<double>(a.inv_freq[i]) * 0.15915494309189533577);  // 1 / (2 pi)
    float sn, cn;
    sincospif(2.0f * static_cast<float>(turns - rint(turns)), &sn, &cn);
    cs[i] = make_float2(cn, sn * a.sign);
  }
}

// Vector indexes of unit u's two vectors; ib < 0: the unit has one vector only.
template <int V, bool INTER>
DSLPG_DEV void unit_vectors(const HeadArgs& a, int u, int& ia, int& ib) {
  if (u < a.rot_units) {
    ia = INTER ? 2 * u : u;
    ib = INTER ? 2 * u + 1 : u + a.rot_units;
  } else {
    ia = 2 * u;  // 2 rot_units + 2 (u - rot_units)
    ib = ia + 1 < a.D / V ? ia + 1 : -1;
  }
}

// Rotate a unit's pairs in place by the angles c[e] = (cos, sin).
template <int V, bool INTER>
DSLPG_DEV void rotate_unit(float (&fa)[V], float (&fb)[V], const float2 (&c)[V], float sgn) {
  if constexpr (INTER) {
#pragma unroll
    for (int e = 0; e < V / 2; ++e) {
      const float2 p = c[e], q = c[V / 2 + e];
      const float a0 = fa[2 * e], a1 = fa[2 * e + 1], b0 = fb[2 * e], b1 = fb[2 * e + 1];
      fa[2 * e] = a0 * p.x - a1 * (p.y * sgn);
      fa[2 * e + 1] = a1 * p.x + a0 * (p.y * sgn);
      fb[2 * e] = b0 * q.x - b1 * (q.y * sgn);
      fb[2 * e + 1] = b1 * q.x + b0 * (q.y * sgn);
    }
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float x0 = fa[e], x1 = fb[e];
      fa[e] = x0 * c[e].x - x1 * (c[e].y * sgn);
      fb[e] = x1 * c[e].x + x0 * (c[e].y * sgn);
    }
  }
}

DSLPG_DEV float lanes_sum(float v, int log_l) {
  for (int k = 0; k < log_l; ++k) v += __shfl_xor_sync(0xffffffffu, v, 1 << k);
  return v;
}

template <typename T, int V, bool INTER, bool NORM>
__global__ void __launch_bounds__(256) heads_fwd_kernel(const HeadArgs a) {
  extern __shared__ __align__(16) float smem_f[];
  float* weights = smem_f;  // [2][D] (NORM)
  float2* table = reinterpret_cast<float2*>(smem_f + (NORM ? 2 * ((a.D + 3) & ~3) : 0));
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  float2* cs = table + static_cast<size_t>(warp) * a.n;
  const int wstride = (a.D + 3) & ~3;
  if constexpr (NORM) {
    for (int i = threadIdx.x; i < 2 * a.D; i += blockDim.x) {
      const int seg = i >= a.D, d = i - seg * a.D;
      weights[seg * wstride + d] = load_any(a.w[seg], d, a.wdt);
    }
    __syncthreads();
  }
  const int u = lane & ((1 << a.log_l) - 1), sub = lane >> a.log_l, rpw = 32 >> a.log_l;
  const bool active = u < a.units;
  int ia = 0, ib = -1;
  if (active) unit_vectors<V, INTER>(a, u, ia, ib);
  const uint32_t items = a.tokens * a.chunks;
  const int all = a.groups[0] + a.groups[1];
  for (uint32_t item = blockIdx.x * warps + warp; item < items; item += gridDim.x * warps) {
    const uint32_t token = item / a.chunks;
    const uint32_t b = token / a.seq, s = token - b * a.seq;
    const int g0 = static_cast<int>((item - token * a.chunks) * a.chunk);
    const int g1 = min(g0 + static_cast<int>(a.chunk), all);
    __syncwarp();
    fill_angles(a, cs, b, s, lane);
    __syncwarp();
    float2 c[V];
#pragma unroll
    for (int e = 0; e < V; ++e) c[e] = (active && u < a.rot_units) ? cs[u * V + e] : make_float2(1.f, 0.f);
    for (int g = g0; g < g1; ++g) {
      const int seg = g >= a.groups[0];
      const int head = (g - seg * a.groups[0]) * rpw + sub;
      const bool ok = active && head < a.heads[seg];
      float fa[V], fb[V];
#pragma unroll
      for (int e = 0; e < V; ++e) fa[e] = fb[e] = 0.f;
      if (ok) {
        const T* src = static_cast<const T*>(a.x[seg]) + b * a.xs[seg][0] + s * a.xs[seg][1] + head * a.xs[seg][2];
        Pack<T, V> p;
        ld_pack(p, src + ia * V);
        unpack_to<T, V>(p, fa);
        if (ib >= 0) {
          ld_pack(p, src + ib * V);
          unpack_to<T, V>(p, fb);
        }
      }
      if constexpr (NORM) {
        float ss = 0.f;
#pragma unroll
        for (int e = 0; e < V; ++e) ss += fa[e] * fa[e] + fb[e] * fb[e];
        const float rstd = rsqrtf(lanes_sum(ss, a.log_l) * a.inv_d + a.eps);
        const float* w = weights + seg * wstride;
#pragma unroll
        for (int e = 0; e < V; ++e) {
          fa[e] *= rstd * w[ia * V + e];
          if (ib >= 0) fb[e] *= rstd * w[ib * V + e];
        }
      }
      if (ok) {
        if (u < a.rot_units) rotate_unit<V, INTER>(fa, fb, c, 1.f);
        T* dst = static_cast<T*>(a.y[seg]) + (static_cast<int64_t>(token) * a.heads[seg] + head) * a.D;
        st_pack<T, V>(dst + ia * V, fa);
        if (ib >= 0) st_pack<T, V>(dst + ib * V, fb);
      }
    }
  }
}

// Norm backward: the first q_ctas CTAs walk q's rows, the others k's, so a
// lane's dw sums (one unit of one weight vector) stay in registers for the
// whole kernel; they are merged over the CTA in a fixed order into one [D] row
// of `partial`, which heads_dw_kernel sums over the CTAs, so that the same
// call gives the same bits.
template <typename T, int V, bool INTER>
__global__ void __launch_bounds__(256) heads_bwd_kernel(const HeadArgs a) {
  extern __shared__ __align__(16) float smem_f[];
  const int wstride = (a.D + 3) & ~3;
  float* weights = smem_f;                                        // [D]
  float* sums = smem_f + wstride;                                 // [warps][D]
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  float2* cs = reinterpret_cast<float2*>(sums + static_cast<size_t>(warps) * wstride) + static_cast<size_t>(warp) * a.n;
  const int seg = static_cast<int>(blockIdx.x) >= a.q_ctas;
  const uint32_t cta = blockIdx.x - (seg ? a.q_ctas : 0), ctas = seg ? gridDim.x - a.q_ctas : a.q_ctas;
  for (int d = threadIdx.x; d < a.D; d += blockDim.x) weights[d] = load_any(a.w[seg], d, a.wdt);
  __syncthreads();
  const int u = lane & ((1 << a.log_l) - 1), sub = lane >> a.log_l, rpw = 32 >> a.log_l;
  const bool active = u < a.units;
  int ia = 0, ib = -1;
  if (active) unit_vectors<V, INTER>(a, u, ia, ib);
  const uint32_t chunk = seg ? a.chunk_k : a.chunk, chunks = seg ? a.chunks_k : a.chunks;
  const uint32_t items = a.tokens * chunks;
  float da[V], db[V];
#pragma unroll
  for (int e = 0; e < V; ++e) da[e] = db[e] = 0.f;
  for (uint32_t item = cta * warps + warp; item < items; item += ctas * warps) {
    const uint32_t token = item / chunks;
    const uint32_t b = token / a.seq, s = token - b * a.seq;
    const int g0 = static_cast<int>((item - token * chunks) * chunk);
    const int g1 = min(g0 + static_cast<int>(chunk), a.groups[seg]);
    __syncwarp();
    fill_angles(a, cs, b, s, lane);
    __syncwarp();
    float2 c[V];
#pragma unroll
    for (int e = 0; e < V; ++e) c[e] = (active && u < a.rot_units) ? cs[u * V + e] : make_float2(1.f, 0.f);
    for (int g = g0; g < g1; ++g) {
      const int head = g * rpw + sub;
      const bool ok = active && head < a.heads[seg];
      float xa[V], xb[V], ga[V], gb[V];
#pragma unroll
      for (int e = 0; e < V; ++e) xa[e] = xb[e] = ga[e] = gb[e] = 0.f;
      if (ok) {
        const T* src = static_cast<const T*>(a.x[seg]) + b * a.xs[seg][0] + s * a.xs[seg][1] + head * a.xs[seg][2];
        const T* dsrc = static_cast<const T*>(a.dy[seg]) + b * a.dys[seg][0] + s * a.dys[seg][1] + head * a.dys[seg][2];
        Pack<T, V> p, q;
        ld_pack(p, src + ia * V);
        ld_pack(q, dsrc + ia * V);
        unpack_to<T, V>(p, xa);
        unpack_to<T, V>(q, ga);
        if (ib >= 0) {
          ld_pack(p, src + ib * V);
          ld_pack(q, dsrc + ib * V);
          unpack_to<T, V>(p, xb);
          unpack_to<T, V>(q, gb);
        }
        if (u < a.rot_units) rotate_unit<V, INTER>(ga, gb, c, 1.f);
      }
      float wa[V], wb[V], ss = 0.f, cc = 0.f;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        wa[e] = weights[ia * V + e];
        wb[e] = ib >= 0 ? weights[ib * V + e] : 0.f;
        ss += xa[e] * xa[e] + xb[e] * xb[e];
        cc += wa[e] * ga[e] * xa[e] + wb[e] * gb[e] * xb[e];
      }
      ss = lanes_sum(ss, a.log_l);
      cc = lanes_sum(cc, a.log_l);
      const float rstd = rsqrtf(ss * a.inv_d + a.eps);
      const float k = rstd * rstd * (cc * a.inv_d);
      if (ok) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
          da[e] += ga[e] * (xa[e] * rstd);
          db[e] += gb[e] * (xb[e] * rstd);
          ga[e] = rstd * (wa[e] * ga[e] - xa[e] * k);
          gb[e] = rstd * (wb[e] * gb[e] - xb[e] * k);
        }
        T* dst = static_cast<T*>(a.y[seg]) + (static_cast<int64_t>(token) * a.heads[seg] + head) * a.D;
        st_pack<T, V>(dst + ia * V, ga);
        if (ib >= 0) st_pack<T, V>(dst + ib * V, gb);
      }
    }
  }
#pragma unroll
  for (int e = 0; e < V; ++e) {
    for (int o = 1 << a.log_l; o < 32; o <<= 1) {
      da[e] += __shfl_xor_sync(0xffffffffu, da[e], o);
      db[e] += __shfl_xor_sync(0xffffffffu, db[e], o);
    }
    if (active && sub == 0) {
      sums[warp * wstride + ia * V + e] = da[e];
      if (ib >= 0) sums[warp * wstride + ib * V + e] = db[e];
    }
  }
  __syncthreads();
  for (int d = threadIdx.x; d < a.D; d += blockDim.x) {
    float t = 0.f;
    for (int k = 0; k < warps; ++k) t += sums[k * wstride + d];
    a.partial[static_cast<int64_t>(blockIdx.x) * a.D + d] = t;
  }
}

// dw[seg][d] = the sum of the CTAs' partial rows: 8 threads a column, each every 8th row, merged in order.
__global__ void __launch_bounds__(256) heads_dw_kernel(const float* partial, int q_ctas, int ctas, int D, float* dq,
                                                       float* dk) {
  __shared__ float part[8][32];
  const int col = threadIdx.x & 31, row = threadIdx.x >> 5;
  const int d = blockIdx.x * 32 + col, seg = blockIdx.y;
  const int lo = seg ? q_ctas : 0, hi = seg ? ctas : q_ctas;
  float t = 0.f;
  if (d < D)
    for (int r = lo + row; r < hi; r += 8) t += partial[static_cast<int64_t>(r) * D + d];
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
__global__ void __launch_bounds__(128) heads_any_kernel(const HeadArgs a) {
  extern __shared__ __align__(16) float smem_f[];
  const int wstride = (a.D + 3) & ~3;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  float* sums = smem_f + warp * wstride;  // BWD: [warps][D]
  float2* cs = reinterpret_cast<float2*>(smem_f + (BWD ? warps * wstride : 0)) + static_cast<size_t>(warp) * a.n;
  const int seg0 = BWD && static_cast<int>(blockIdx.x) >= a.q_ctas;
  const uint32_t cta = blockIdx.x - (seg0 ? a.q_ctas : 0);
  const uint32_t ctas = BWD ? (seg0 ? gridDim.x - a.q_ctas : a.q_ctas) : gridDim.x;
  const int first = BWD ? (seg0 ? a.heads[0] : 0) : 0;
  const int count = BWD ? a.heads[seg0] : a.heads[0] + a.heads[1];
  const uint32_t chunk = seg0 ? a.chunk_k : a.chunk, chunks = seg0 ? a.chunks_k : a.chunks;
  if constexpr (BWD)
    for (int d = lane; d < a.D; d += 32) sums[d] = 0.f;
  const int n = a.n, D = a.D;
  // Index of the two members of pair i.
  auto lo = [&](int i) { return a.interleaved ? 2 * i : i; };
  auto hi = [&](int i) { return a.interleaved ? 2 * i + 1 : i + n; };
  const uint32_t items = a.tokens * chunks;
  for (uint32_t item = cta * warps + warp; item < items; item += ctas * warps) {
    const uint32_t token = item / chunks;
    const uint32_t b = token / a.seq, s = token - b * a.seq;
    const int h0 = static_cast<int>((item - token * chunks) * chunk);
    const int h1 = min(h0 + static_cast<int>(chunk), count);
    __syncwarp();
    fill_angles(a, cs, b, s, lane);
    __syncwarp();
    for (int h = first + h0; h < first + h1; ++h) {
      const int seg = h >= a.heads[0], head = h - (seg ? a.heads[0] : 0);
      const T* src = static_cast<const T*>(a.x[seg]) + b * a.xs[seg][0] + s * a.xs[seg][1] + head * a.xs[seg][2];
      T* dst = static_cast<T*>(a.y[seg]) + (static_cast<int64_t>(token) * a.heads[seg] + head) * D;
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
          sums[d] += g * (v * rstd);  // feature d is the same lane's in every row
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
    for (int d = threadIdx.x; d < D; d += blockDim.x) {
      float t = 0.f;
      for (int k = 0; k < warps; ++k) t += smem_f[k * wstride + d];
      a.partial[static_cast<int64_t>(blockIdx.x) * D + d] = t;
    }
  }
}

namespace {

constexpr int kMaxHeadDim = 1024;
constexpr int kPartialRows = 1184;  // CTAs of a norm backward at most (8 for each of 148 SMs)

// Groups of heads a warp takes per item: all of a token's, fewer while that leaves warps without work.
uint32_t chunk_of(int groups, uint32_t tokens, int64_t warps) {
  int64_t chunk = groups;
  while (chunk > 1 && static_cast<int64_t>(tokens) * ((groups + chunk - 1) / chunk) < warps) chunk = (chunk + 1) / 2;
  return static_cast<uint32_t>(chunk < 1 ? 1 : chunk);
}

template <typename K>
int grid_for(K kernel, int block, size_t smem, int64_t items, cudaError_t& e) {
  const void* fn = reinterpret_cast<const void*>(kernel);
  if (smem > 48 * 1024 && (e = allow_dynamic_smem(fn, smem)) != cudaSuccess) return 0;
  return persistent_grid(fn, block, smem, (items + block / 32 - 1) / (block / 32));
}

// The q : k split of a norm backward's CTAs, by their groups.
int split_ctas(const HeadArgs& a, int grid) {
  const int64_t all = a.groups[0] + a.groups[1];
  if (a.groups[1] == 0) return grid;
  int64_t q = (static_cast<int64_t>(grid) * a.groups[0] + all / 2) / all;
  if (a.groups[0] > 0 && q < 1) q = 1;
  if (q > grid - 1) q = grid - 1;
  return static_cast<int>(q);
}

template <typename T, int V, bool INTER, bool NORM>
cudaError_t launch_fwd(HeadArgs a, cudaStream_t st) {
  const int block = 256;
  const size_t smem = (NORM ? 2 * ((a.D + 3) & ~3) * 4 : 0) + static_cast<size_t>(block / 32) * a.n * 8;
  const int all = a.groups[0] + a.groups[1];
  a.chunk = chunk_of(all, a.tokens, static_cast<int64_t>(sm_count()) * 16);
  a.chunks = (all + a.chunk - 1) / a.chunk;
  cudaError_t e = cudaSuccess;
  const int grid = grid_for(&heads_fwd_kernel<T, V, INTER, NORM>, block, smem, static_cast<int64_t>(a.tokens) * a.chunks, e);
  if (e != cudaSuccess) return e;
  heads_fwd_kernel<T, V, INTER, NORM><<<grid, block, smem, st>>>(a);
  return cudaGetLastError();
}

template <typename K>
cudaError_t launch_bwd_with(K kernel, HeadArgs a, int block, size_t smem, float* dwq, float* dwk, cudaStream_t st) {
  const int64_t want = static_cast<int64_t>(sm_count()) * 16;
  a.chunk = chunk_of(a.groups[0], a.tokens, want);
  a.chunks = (a.groups[0] + a.chunk - 1) / a.chunk;
  a.chunk_k = chunk_of(a.groups[1], a.tokens, want);
  a.chunks_k = (a.groups[1] + a.chunk_k - 1) / a.chunk_k;
  cudaError_t e = cudaSuccess;
  int grid = grid_for(kernel, block, smem, static_cast<int64_t>(a.tokens) * (a.chunks + a.chunks_k), e);
  if (e != cudaSuccess) return e;
  if (grid > kPartialRows) grid = kPartialRows;
  if (grid < 2) grid = 2;
  a.q_ctas = split_ctas(a, grid);
  kernel<<<grid, block, smem, st>>>(a);
  if ((e = cudaGetLastError()) != cudaSuccess) return e;
  heads_dw_kernel<<<dim3((a.D + 31) / 32, 2), 256, 0, st>>>(a.partial, a.q_ctas, grid, a.D, dwq, dwk);
  return cudaGetLastError();
}

template <typename T, int V, bool INTER>
cudaError_t launch_bwd(HeadArgs a, float* dwq, float* dwk, cudaStream_t st) {
  const int block = 256, ws = (a.D + 3) & ~3;
  const size_t smem = static_cast<size_t>(ws) * 4 * (1 + block / 32) + static_cast<size_t>(block / 32) * a.n * 8;
  return launch_bwd_with(&heads_bwd_kernel<T, V, INTER>, a, block, smem, dwq, dwk, st);
}

template <typename T, bool NORM, bool BWD>
cudaError_t launch_any(HeadArgs a, float* dwq, float* dwk, cudaStream_t st) {
  const int block = 128, ws = (a.D + 3) & ~3;
  const size_t smem = (BWD ? static_cast<size_t>(ws) * 4 * (block / 32) : 0) + static_cast<size_t>(block / 32) * a.n * 8;
  a.groups[0] = a.heads[0];
  a.groups[1] = a.heads[1];
  if constexpr (BWD) {
    return launch_bwd_with(&heads_any_kernel<T, NORM, true>, a, block, smem, dwq, dwk, st);
  } else {
    const int all = a.heads[0] + a.heads[1];
    a.chunk = chunk_of(all, a.tokens, static_cast<int64_t>(sm_count()) * 16);
    a.chunks = (all + a.chunk - 1) / a.chunk;
    cudaError_t e = cudaSuccess;
    const int grid =
        grid_for(&heads_any_kernel<T, NORM, false>, block, smem, static_cast<int64_t>(a.tokens) * a.chunks, e);
    if (e != cudaSuccess) return e;
    heads_any_kernel<T, NORM, false><<<grid, block, smem, st>>>(a);
    return cudaGetLastError();
  }
}

// Whether rows can be cut into units of two V-element vectors: sizes, strides and bases.
template <typename T>
bool fits(const HeadArgs& a, int V, bool bwd) {
  if (a.D % V || a.n % V) return false;  // n % V: half of the rotated features, or 2 V of them interleaved
  const int units = a.n / V + (a.D / V - 2 * (a.n / V) + 1) / 2;
  if (units > 32) return false;
  const int bytes = V * static_cast<int>(sizeof(T));
  for (int seg = 0; seg < 2; ++seg) {
    if (!aligned(a.x[seg], bytes) || !aligned(a.y[seg], bytes) || (bwd && !aligned(a.dy[seg], bytes))) return false;
    for (int k = 0; k < 3; ++k)
      if (a.xs[seg][k] % V || (bwd && a.dys[seg][k] % V)) return false;
  }
  return true;
}

void set_units(HeadArgs& a, int V) {
  a.rot_units = a.n / V;
  a.units = a.rot_units + (a.D / V - 2 * a.rot_units + 1) / 2;
  a.log_l = 0;
  while ((1 << a.log_l) < a.units) ++a.log_l;
  const int rpw = 32 >> a.log_l;
  for (int seg = 0; seg < 2; ++seg) a.groups[seg] = (a.heads[seg] + rpw - 1) / rpw;
}

template <typename T, int V, bool INTER>
cudaError_t launch_v(HeadArgs a, bool norm, bool bwd, float* dwq, float* dwk, cudaStream_t st) {
  set_units(a, V);
  if (bwd) return launch_bwd<T, V, INTER>(a, dwq, dwk, st);
  return norm ? launch_fwd<T, V, INTER, true>(a, st) : launch_fwd<T, V, INTER, false>(a, st);
}

template <typename T>
cudaError_t dispatch(HeadArgs a, bool norm, bool bwd, float* dwq, float* dwk, cudaStream_t st) {
  constexpr int E = Elt<T>::kPerVec;
  if (kernel_path() != DSLPG_PATH_STREAM) {
    if (fits<T>(a, E, bwd))
      return a.interleaved ? launch_v<T, E, true>(a, norm, bwd, dwq, dwk, st)
                           : launch_v<T, E, false>(a, norm, bwd, dwq, dwk, st);
    if (fits<T>(a, E / 2, bwd))
      return a.interleaved ? launch_v<T, E / 2, true>(a, norm, bwd, dwq, dwk, st)
                           : launch_v<T, E / 2, false>(a, norm, bwd, dwq, dwk, st);
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
  *bytes = kPartialRows * head_dim * 4;
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
  if (workspace_bytes < static_cast<int64_t>(kPartialRows) * a.D * 4 || !aligned(workspace, 16)) return DSLPG_ERR_BAD_ARGUMENT;
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
