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
// of them.  Angles are turns in double (position times frequency, less the nearest whole number) until
// sincospi: a float32 angle would be off by 0.06 at position 10^6.
//
// p[]: [0] B, [1] T, [2] H, [3] flags, [4] head groups of a block (a power of two), [5] parts of the batch,
// [6] eps (float bits), [7] log2(base) / (TCB_ROT / 2) (double bits).  dgain's partial sums go to scratch.
#pragma once

namespace tcb {

constexpr u32 HN_SHARED = 1, HN_HEADS_FIRST = 2, HN_DX = 4, HN_DGAIN = 8;
constexpr int HN_PAIRS = TCB_ROT / 2;

constexpr int hn_pow2(int x) {
  int p = 1;
  while (p < x) p *= 2;
  return p;
}
// A row as units of 2 V values: first the pairs, V at a time, then the rest of the head.
template <int V> struct HnRow {
  static constexpr int PU = (HN_PAIRS + V - 1) / V, RU = (TCB_D - TCB_ROT + 2 * V - 1) / (2 * V);
  static constexpr int U = PU + RU;
  static constexpr int LANES = hn_pow2(U) < 32 ? hn_pow2(U) : 32;
  static constexpr int PER = (U + LANES - 1) / LANES;   // units a lane
  static constexpr int GROUPS = 256 / LANES;

  // A unit's values: pairs' first members (or the first V of the rest) in a, the others in b.
  __device__ static void load(const float* row, int u, float (&a)[V], float (&b)[V]) {
#pragma unroll
    for (int j = 0; j < V; ++j) a[j] = b[j] = 0.0f;
    if (u < PU) {
      if (TCB_INTERLEAVED) {
        float q[2 * V];
        tcb::load<V>(*reinterpret_cast<float(*)[V]>(&q[0]), row + 2 * V * u);
        tcb::load<V>(*reinterpret_cast<float(*)[V]>(&q[V]), row + 2 * V * u + V);
#pragma unroll
        for (int j = 0; j < V; ++j) { a[j] = q[2 * j]; b[j] = q[2 * j + 1]; }
      } else {
        tcb::load<V>(a, row + V * u);
        tcb::load<V>(b, row + HN_PAIRS + V * u);
      }
    } else if (u < U) {
      const int c = TCB_ROT + 2 * V * (u - PU);
      tcb::load<V>(a, row + c);
      if (c + V < TCB_D) tcb::load<V>(b, row + c + V);
    }
  }
  __device__ static void store(float* row, int u, const float (&a)[V], const float (&b)[V]) {
    if (u < PU) {
      if (TCB_INTERLEAVED) {
        float q[2 * V];
#pragma unroll
        for (int j = 0; j < V; ++j) { q[2 * j] = a[j]; q[2 * j + 1] = b[j]; }
        tcb::store<V>(row + 2 * V * u, *reinterpret_cast<float(*)[V]>(&q[0]));
        tcb::store<V>(row + 2 * V * u + V, *reinterpret_cast<float(*)[V]>(&q[V]));
      } else {
        tcb::store<V>(row + V * u, a);
        tcb::store<V>(row + HN_PAIRS + V * u, b);
      }
    } else if (u < U) {
      const int c = TCB_ROT + 2 * V * (u - PU);
      tcb::store<V>(row + c, a);
      if (c + V < TCB_D) tcb::store<V>(row + c + V, b);
    }
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
  const u32 B = (u32)a.p[0], T = (u32)a.p[1], H = (u32)a.p[2], flags = (u32)a.p[3], parts = (u32)a.p[5];
  const u32 HG = (u32)a.p[4] < (u32)R::GROUPS ? (u32)a.p[4] : (u32)R::GROUPS;
  const float eps = __uint_as_float((u32)a.p[6]);
  const bool first = (flags & HN_HEADS_FIRST) != 0, shared = (flags & HN_SHARED) != 0;
  const float* x = reinterpret_cast<const float*>(a.in[0]);
  const float* gy = reinterpret_cast<const float*>(a.in[3]);
  float* out = reinterpret_cast<float*>(a.out);
  // frequencies in turns a position
  for (int i = threadIdx.x; i < HN_PAIRS; i += 256)
    inv[i] = exp2(-(double)i * __longlong_as_double(a.p[7])) * 0.15915494309189535;
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
  const u32 tiles = (T + TT - 1) / TT, units = tiles * parts;
  for (u32 u = blockIdx.x; u < units; u += gridDim.x) {
    // every lane of a warp takes part in the sums, so a group without a token or a head only does not store
    const u32 tt = (u % tiles) * TT + tg, t = tt < T ? tt : T - 1;
    const u32 part = u / tiles, b1 = (u32)((u64)(part + 1) * B / parts);
    float c[R::PER][V], s[R::PER][V];
    bool known = false;
    for (u32 b = (u32)((u64)part * B / parts); b < b1; ++b) {
      if (HN_PAIRS > 0 && !(known && shared)) {
        const double pos = (double)ld1(reinterpret_cast<const float*>(a.in[2]) + (shared ? 0 : (u64)b * T) + t);
#pragma unroll
        for (int k = 0; k < R::PER; ++k)
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const int i = (lane + k * R::LANES) * V + j;
            c[k][j] = 1.0f;
            s[k][j] = 0.0f;
            if (i < HN_PAIRS) {
              const double turn = pos * inv[i];
              sincospif(2.0f * (float)(turn - rint(turn)), &s[k][j], &c[k][j]);
            }
          }
        known = true;
      }
      for (u32 h0 = 0; h0 < H; h0 += HG) {
        const u32 hh = h0 + hg, h = hh < H ? hh : H - 1;
        const bool mine = hh < H && tt < T;
        const u64 src = (((u64)b * T + t) * H + h) * TCB_D;
        const u64 dst = first ? (((u64)b * H + h) * T + t) * TCB_D : src;
        float xa[R::PER][V], xb[R::PER][V];
        float ss = 0.0f;
#pragma unroll
        for (int k = 0; k < R::PER; ++k) R::load(x + src, lane + k * R::LANES, xa[k], xb[k]);
        if (!BACK) {
#pragma unroll
          for (int k = 0; k < R::PER; ++k)
#pragma unroll
            for (int j = 0; j < V; ++j) ss += xa[k][j] * xa[k][j] + xb[k][j] * xb[k][j];
          const float r = 1.0f / sqrtf(group_sum<R::LANES>(ss) * (1.0f / TCB_D) + eps);
          if (!mine) continue;
#pragma unroll
          for (int k = 0; k < R::PER; ++k) {
            const int un = lane + k * R::LANES;
#pragma unroll
            for (int j = 0; j < V; ++j) {
              const float p = xa[k][j] * r * ga[k][j], q = xb[k][j] * r * gb[k][j];
              const bool turn = HN_PAIRS > 0 && un < R::PU;
              xa[k][j] = turn ? p * c[k][j] - q * s[k][j] : p;
              xb[k][j] = turn ? q * c[k][j] + p * s[k][j] : q;
            }
            R::store(out + dst, un, xa[k], xb[k]);
          }
        } else {
          float ua[R::PER][V], ub[R::PER][V];
          float dot = 0.0f;
#pragma unroll
          for (int k = 0; k < R::PER; ++k) R::load(gy + dst, lane + k * R::LANES, ua[k], ub[k]);
#pragma unroll
          for (int k = 0; k < R::PER; ++k)
#pragma unroll
            for (int j = 0; j < V; ++j) {
              if (HN_PAIRS > 0 && lane + k * R::LANES < R::PU) {
                const float p = ua[k][j], q = ub[k][j];
                ua[k][j] = p * c[k][j] + q * s[k][j];
                ub[k][j] = q * c[k][j] - p * s[k][j];
              }
              ss += xa[k][j] * xa[k][j] + xb[k][j] * xb[k][j];
              dot += ua[k][j] * ga[k][j] * xa[k][j] + ub[k][j] * gb[k][j] * xb[k][j];
            }
          ss = group_sum<R::LANES>(ss);
          dot = group_sum<R::LANES>(dot);
          const float r = 1.0f / sqrtf(ss * (1.0f / TCB_D) + eps);
          const float m = dot * r * r * (1.0f / TCB_D);
          if (!mine) continue;
#pragma unroll
          for (int k = 0; k < R::PER; ++k) {
#pragma unroll
            for (int j = 0; j < V; ++j) {
              da[k][j] += ua[k][j] * xa[k][j] * r;
              db[k][j] += ub[k][j] * xb[k][j] * r;
              xa[k][j] = r * (ua[k][j] * ga[k][j] - xa[k][j] * m);
              xb[k][j] = r * (ub[k][j] * gb[k][j] - xb[k][j] * m);
            }
            if (flags & HN_DX) R::store(out + src, lane + k * R::LANES, xa[k], xb[k]);
          }
        }
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

extern "C" __global__ void __launch_bounds__(256) tcb_head_norm_rope(const tcb::Args a) {
  tcb::grid_dependency_sync();
  if constexpr (tcb::HN_WIDE) {
    if (((a.in[0] | a.in[1] | a.out) & 15) == 0) return tcb::head_norm_rope<4, false>(a);
  }
  tcb::head_norm_rope<1, false>(a);
}

extern "C" __global__ void __launch_bounds__(256) tcb_head_norm_rope_grad(const tcb::Args a) {
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
  if (col < TCB_D) {
#pragma unroll 10
    for (u32 k = row; k < (u32)a.p[0]; k += 128) s += p[(u64)k * TCB_D + col];
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
