// tcb/head_norm_rope.cuh -- RMS norm of every head, rotation by position and the move of the head axis in
// front of the tokens, in one pass over the values, and its gradients (the IR ops headNormRope and
// headNormRopeGrad).
//
//   x [B, T, H, D], gain [D], pos [T] or [B, T]
//   n = x r gain,  r = 1 / sqrt(mean_D x^2 + eps)
//   y = n with each of its first TCB_ROT / 2 pairs turned by pos * base^(-2i / TCB_ROT): pair i is
//       (n_i, n_i+TCB_ROT/2), or (n_2i, n_2i+1) with TCB_INTERLEAVED; the rest of the head as it is
//   y [B, H, T, D] (what attention reads), or [B, T, H, D]
// Backward, u = y's cotangent turned back: dgain = sum u x r,  dx = r (u gain - x r^2 mean(u gain x)).
//
// Bound by memory: 8 bytes a value forward, 12 backward, each read or written once.  A group of lanes
// holds a row in registers, both halves of a pair in the same lane, and walks the heads (and, where the
// positions are shared, the batch) of one token, so an angle's sine and cosine are computed once for all
// of them; the next row is on its way while one is worked on.  Every CTA of one full wave takes an equal run
// of the steps (token tile, batch, head group; 4 % uneven at 512 x 256 x 4 x 64, where whole tiles left a
// second, partial wave).  Angles are turns in double (position times frequency, less the nearest whole number) until
// sincospi: a float32 angle would be off by 0.06 at position 10^6.
//
// p[]: [0] B, [1] T, [2] H, [3] flags, [4] heads of a block (a power of two), [5] eps (float bits), [6]
// log2(base) / (TCB_ROT / 2) (double bits).  dgain's partial sums go to scratch.
#pragma once

namespace tcb {

constexpr u32 HN_SHARED = 1, HN_HEADS_FIRST = 2, HN_DX = 4, HN_DGAIN = 8;
constexpr int HN_PAIRS = TCB_ROT / 2;

constexpr int hn_pow2(int x) {
  int p = 1;
  while (p < x) p *= 2;
  return p;
}
// A row as units of 2 V values: first the pairs, V at a time, then the rest of the head.  (V is 1, or 4 where
// HN_WIDE holds: then PU counts whole units.)
template <int V> struct HnRow {
  static constexpr int PU = (HN_PAIRS + V - 1) / V, RU = (TCB_D - TCB_ROT + 2 * V - 1) / (2 * V);
  static constexpr int U = PU + RU;
  static constexpr int LANES = hn_pow2(U) < 32 ? hn_pow2(U) : 32;
  static constexpr int PER = (U + LANES - 1) / LANES;   // units a lane
  static constexpr int GROUPS = 256 / LANES;

  // Where a unit's two runs of V values begin: the halves of its pairs (interleaved: two runs of whole pairs,
  // half the turned part apart; of the rest likewise), so that neighbouring lanes read and write neighbours.
  static constexpr bool SPLIT = TCB_INTERLEAVED && V > 1;
  __device__ static int at(int u, bool second) {
    if (u < PU) return TCB_INTERLEAVED && V == 1 ? 2 * u + second : V * u + (second ? HN_PAIRS : 0);
    return TCB_ROT + V * (u - PU + (second ? RU : 0));
  }
  // which pair the unit's j-th is
  __device__ static int pair(int u, int j) {
    return SPLIT ? V / 2 * u + j % (V / 2) + (j < V / 2 ? 0 : HN_PAIRS / 2) : V * u + j;
  }

  // A unit's values: pairs' first members (or the first run of the rest) in a, the others in b.
  __device__ static void load(const float* row, int u, float (&a)[V], float (&b)[V]) {
#pragma unroll
    for (int j = 0; j < V; ++j) a[j] = b[j] = 0.0f;
    if (u >= U) return;
    tcb::load<V>(a, row + at(u, false));
    if (u < PU || at(u, true) < TCB_D) tcb::load<V>(b, row + at(u, true));
    if constexpr (SPLIT)
      if (u < PU) {   // (p0 q0 p1 q1) (p2 q2 p3 q3) to (p0 p1 p2 p3) (q0 q1 q2 q3)
        const float q[8] = {a[0], a[2], b[0], b[2], a[1], a[3], b[1], b[3]};
#pragma unroll
        for (int j = 0; j < 4; ++j) { a[j] = q[j]; b[j] = q[4 + j]; }
      }
  }
  __device__ static void store(float* row, int u, const float (&a)[V], const float (&b)[V]) {
    if (u >= U) return;
    float p[V], q[V];
#pragma unroll
    for (int j = 0; j < V; ++j) { p[j] = a[j]; q[j] = b[j]; }
    if constexpr (SPLIT)
      if (u < PU) {   // and back
        p[1] = b[0]; p[2] = a[1]; p[3] = b[1];
        q[0] = a[2]; q[1] = b[2]; q[2] = a[3];
      }
    tcb::store<V>(row + at(u, false), p);
    if (u < PU || at(u, true) < TCB_D) tcb::store<V>(row + at(u, true), q);
  }
};

template <int LANES>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

template <int V, bool BACK>
__device__ __forceinline__ void head_norm_rope(const Args& a) {
  using R = HnRow<V>;
  __shared__ double inv[HN_PAIRS > 0 ? HN_PAIRS : 1];
  const u32 B = (u32)a.p[0], T = (u32)a.p[1], H = (u32)a.p[2], flags = (u32)a.p[3];
  const u32 HG = (u32)a.p[4] < (u32)R::GROUPS ? (u32)a.p[4] : (u32)R::GROUPS;
  const float eps = __uint_as_float((u32)a.p[5]);
  const bool first = (flags & HN_HEADS_FIRST) != 0, shared = (flags & HN_SHARED) != 0;
  const float* x = reinterpret_cast<const float*>(a.in[0]);
  const float* gy = reinterpret_cast<const float*>(a.in[3]);
  float* out = reinterpret_cast<float*>(a.out);
  // frequencies in turns a position
  for (int i = threadIdx.x; i < HN_PAIRS; i += 256)
    inv[i] = exp2(-(double)i * __longlong_as_double(a.p[6])) * 0.15915494309189535;
  __syncthreads();
  const int lane = threadIdx.x % R::LANES;
  const u32 group = threadIdx.x / R::LANES, hg = group % HG, tg = group / HG, TT = R::GROUPS / HG;
  float ga[R::PER][V], gb[R::PER][V], da[R::PER][V], db[R::PER][V];
#pragma unroll
  for (int k = 0; k < R::PER; ++k) {
    R::load(reinterpret_cast<const float*>(a.in[1]), lane + k * R::LANES, ga[k], gb[k]);
#pragma unroll
    for (int j = 0; j < V; ++j) da[k][j] = db[k][j] = 0.0f;
  }
  // this CTA's run of steps: head groups fastest, then the batch, then the tiles of TT tokens
  const u32 hs = (H + HG - 1) / HG;
  const u64 steps = (u64)((T + TT - 1) / TT) * B * hs;
  const u64 lo = blockIdx.x * steps / gridDim.x, hi = (blockIdx.x + 1) * steps / gridDim.x;
  // every lane of a warp takes part in the sums, so a group without a token or a head only does not store
  struct Row { u32 tile, b, h0; u64 src, dst; bool mine; };
  Row r;
  auto locate = [&](Row& q) {
    const u32 tt = q.tile * TT + tg, hh = q.h0 * HG + hg, t = tt < T ? tt : T - 1, h = hh < H ? hh : H - 1;
    q.mine = tt < T && hh < H;
    q.src = (((u64)q.b * T + t) * H + h) * TCB_D;
    q.dst = first ? (((u64)q.b * H + h) * T + t) * TCB_D : q.src;
  };
  r.tile = (u32)(lo / ((u64)B * hs));
  const u64 in_tile = lo - (u64)r.tile * B * hs;
  r.b = (u32)(in_tile / hs);
  r.h0 = (u32)(in_tile - (u64)r.b * hs);
  locate(r);
  float xa[R::PER][V], xb[R::PER][V], ua[R::PER][V], ub[R::PER][V], c[R::PER][V], s[R::PER][V];
  auto fetch = [&](const Row& q) {
#pragma unroll
    for (int k = 0; k < R::PER; ++k) {
      R::load(x + q.src, lane + k * R::LANES, xa[k], xb[k]);
      if (BACK) R::load(gy + q.dst, lane + k * R::LANES, ua[k], ub[k]);
    }
  };
  if (lo < hi) fetch(r);
  bool turn_angles = true;
  for (u64 i = lo; i < hi; ++i) {
    if (HN_PAIRS > 0 && turn_angles) {
      const u32 tt = r.tile * TT + tg, t = tt < T ? tt : T - 1;
      const double pos = (double)ld1(reinterpret_cast<const float*>(a.in[2]) + (shared ? 0 : (u64)r.b * T) + t);
#pragma unroll
      for (int k = 0; k < R::PER; ++k)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const int un = lane + k * R::LANES, p = R::pair(un, j);
          c[k][j] = 1.0f;
          s[k][j] = 0.0f;
          if (un < R::PU) {
            const double turn = pos * inv[p];
            sincospif(2.0f * (float)(turn - rint(turn)), &s[k][j], &c[k][j]);
          }
        }
    }
    // the row at hand out of the way of the next one
    const Row q = r;
    float ya[R::PER][V], yb[R::PER][V], va[R::PER][V], vb[R::PER][V];
#pragma unroll
    for (int k = 0; k < R::PER; ++k)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        ya[k][j] = xa[k][j];
        yb[k][j] = xb[k][j];
        if (BACK) { va[k][j] = ua[k][j]; vb[k][j] = ub[k][j]; }
      }
    turn_angles = false;
    if (++r.h0 == hs) {
      r.h0 = 0;
      turn_angles = !shared;
      if (++r.b == B) { r.b = 0; ++r.tile; turn_angles = true; }
    }
    if (i + 1 < hi) {
      locate(r);
      fetch(r);
    }
    float ss = 0.0f, dot = 0.0f;
#pragma unroll
    for (int k = 0; k < R::PER; ++k)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        ss += ya[k][j] * ya[k][j] + yb[k][j] * yb[k][j];
        if (BACK) {
          if (HN_PAIRS > 0 && lane + k * R::LANES < R::PU) {
            const float p = va[k][j], w = vb[k][j];
            va[k][j] = p * c[k][j] + w * s[k][j];
            vb[k][j] = w * c[k][j] - p * s[k][j];
          }
          dot += va[k][j] * ga[k][j] * ya[k][j] + vb[k][j] * gb[k][j] * yb[k][j];
        }
      }
    ss = group_sum<R::LANES>(ss);
    if (BACK) dot = group_sum<R::LANES>(dot);
    const float n = 1.0f / sqrtf(ss * (1.0f / TCB_D) + eps);
    if (!q.mine) continue;
    if (!BACK) {
#pragma unroll
      for (int k = 0; k < R::PER; ++k) {
        const int un = lane + k * R::LANES;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float p = ya[k][j] * n * ga[k][j], w = yb[k][j] * n * gb[k][j];
          const bool turn = HN_PAIRS > 0 && un < R::PU;
          ya[k][j] = turn ? p * c[k][j] - w * s[k][j] : p;
          yb[k][j] = turn ? w * c[k][j] + p * s[k][j] : w;
        }
        R::store(out + q.dst, un, ya[k], yb[k]);
      }
    } else {
      const float m = dot * n * n * (1.0f / TCB_D);
#pragma unroll
      for (int k = 0; k < R::PER; ++k) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          da[k][j] += va[k][j] * ya[k][j] * n;
          db[k][j] += vb[k][j] * yb[k][j] * n;
          ya[k][j] = n * (va[k][j] * ga[k][j] - ya[k][j] * m);
          yb[k][j] = n * (vb[k][j] * gb[k][j] - yb[k][j] * m);
        }
        if (flags & HN_DX) R::store(out + q.src, lane + k * R::LANES, ya[k], yb[k]);
      }
    }
  }
  if (BACK && (flags & HN_DGAIN)) {
    // this block's share of dgain: the groups' sums added in group order
    extern __shared__ __align__(16) float acc[];   // [GROUPS][TCB_D]
#pragma unroll
    for (int k = 0; k < R::PER; ++k) R::store(acc + group * TCB_D, lane + k * R::LANES, da[k], db[k]);
    __syncthreads();
    for (int i = threadIdx.x; i < TCB_D; i += 256) {
      float v = 0.0f;
      for (int g = 0; g < R::GROUPS; ++g) v += acc[g * TCB_D + i];
      reinterpret_cast<float*>(a.scratch)[(u64)blockIdx.x * TCB_D + i] = v;
    }
  }
}

// 128-bit lanes where every piece of a row starts on 16 bytes
constexpr bool HN_WIDE = HN_PAIRS % 4 == 0 && TCB_D % 4 == 0;

}  // namespace tcb

extern "C" __global__ void __launch_bounds__(256, 4) tcb_head_norm_rope(const tcb::Args a) {
  tcb::grid_dependency_sync();
  if constexpr (tcb::HN_WIDE) {
    if (((a.in[0] | a.in[1] | a.out) & 15) == 0) return tcb::head_norm_rope<4, false>(a);
  }
  tcb::head_norm_rope<1, false>(a);
}

extern "C" __global__ void __launch_bounds__(256, 2) tcb_head_norm_rope_grad(const tcb::Args a) {
  tcb::grid_dependency_sync();
  if constexpr (tcb::HN_WIDE) {
    if (((a.in[0] | a.in[1] | a.in[3] | a.out) & 15) == 0) return tcb::head_norm_rope<4, true>(a);
  }
  tcb::head_norm_rope<1, true>(a);
}

// dgain: the blocks' shares added up, 8 columns a block; thread row k takes the shares k, k + 128, ...
// p[0]: the shares.
extern "C" __global__ void __launch_bounds__(1024) tcb_head_gain_finish(const tcb::Args a) {
  tcb::grid_dependency_sync();
  __shared__ float sh[32][8];
  const int c = threadIdx.x & 7, row = threadIdx.x >> 3, col = blockIdx.x * 8 + c;
  const float* p = reinterpret_cast<const float*>(a.scratch);
  float s = 0.0f;
  const u32 n = (u32)a.p[0];
#pragma unroll
  for (u32 k = 0; k < 5; ++k) {   // at most 4 CTAs an SM left a share: all loads in flight
    const u32 i = row + 128 * k;
    s += i < n && col < TCB_D ? __ldcg(p + (u64)i * TCB_D + col) : 0.0f;
  }
  s += __shfl_xor_sync(0xffffffffu, s, 8);
  s += __shfl_xor_sync(0xffffffffu, s, 16);
  if ((threadIdx.x & 31) < 8) sh[threadIdx.x >> 5][c] = s;
  __syncthreads();
  if (threadIdx.x < 8 && col < TCB_D) {
    s = 0.0f;
#pragma unroll
    for (int k = 0; k < 32; ++k) s += sh[k][c];
    reinterpret_cast<float*>(a.out)[col] = s;
  }
}
