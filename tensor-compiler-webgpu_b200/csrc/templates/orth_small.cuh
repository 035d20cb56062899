// tcb/orth_small.cuh -- Newton-Schulz orthogonalisation (tcb/orthogonalize.cuh) of matrices that fit one SM:
// a short side of at most TCB_ROWS (64 or 128), a long one of at most TCB_COLS.
//
// One CTA a matrix, one launch.  Bound by latency: 15 dependent products, each about a microsecond of
// issue, tensor core and epilogue (as launches of their own they took 3.5 us each: 64 x 64, 62 us in all).
// X (wide; a tall matrix is held transposed), S and P stay in shared memory as fp16 hi / lo, in blocks of
// 64 columns: rows of 128 bytes in the 128-byte swizzle, which the tensor core reads along the rows (X X^T,
// S S, P) and across them (X in P X) alike.  Rows beyond the short side and columns beyond the long one are
// zero; what the 128-row instruction reads below TCB_ROWS only makes rows that nobody looks at.
//
// grid: matrices; in[0] -> out; p[0] m, p[1] n, p[2] steps, p[15] the error word.  No block looks at the word: only
// a wait of 2 s that ran out writes it.  In scratch, at its start, it holds what other launches left, and the first
// block clears it; a resident program's own word stays until it is read.
#pragma once
#include "tcb/gemm_f16x3.cuh"

namespace tcb {

constexpr u32 OS_PLANE = TCB_ROWS * 128, OS_BLOCK = 2 * OS_PLANE;   // bytes; hi plane, lo plane
constexpr u32 OS_XB = TCB_COLS / 64, OS_SB = TCB_ROWS / 64;         // blocks of X, of S and P
constexpr u32 OS_BYTES = (OS_XB + 2 * OS_SB) * OS_BLOCK + 16384;    // the last 128 rows may be read past the end

// byte offset of the 16-byte chunk (8 columns) holding column c of row r
__device__ __forceinline__ u32 os_at(u32 r, u32 c) { return (c >> 6) * OS_BLOCK + r * 128 + ((((c >> 3) & 7) ^ (r & 7)) << 4); }

template <bool MN> __device__ __forceinline__ u32 os_lo(u32 addr) { return (addr >> 4) | (MN ? OS_BLOCK >> 4 : 1) << 16; }
constexpr u32 OS_HI = 1024u >> 4 | 1u << 14 | 2u << 29;   // 8-row groups 1 KB apart, 128-byte swizzle

// `steps` K steps of 16, A along its rows from block a, B along its rows or (BMN) across them, three
// accumulators of ACC columns (0: one).
template <u32 N, bool BMN, u32 ACC>
__device__ __forceinline__ void os_product(u32 tmem, u32 a, u32 b, u32 steps) {
  constexpr u32 ID = idesc_f16(128, N, 0, BMN ? 1 : 0), L = OS_PLANE >> 4;
  for (u32 k = 0; k < steps; ++k) {
    const u32 ka = (k >> 2) * OS_BLOCK + (k & 3) * 32;
    const u32 ah = os_lo<false>(a + ka), bh = os_lo<BMN>(b + (BMN ? k * 2048 : ka));
    mma_f16<1, ID, OS_HI, OS_HI>(tmem + (ACC ? ACC : 0), ah + L, bh, k != 0);
    mma_f16<1, ID, OS_HI, OS_HI>(tmem + 2 * ACC, ah, bh + L, ACC ? k != 0 : true);
    mma_f16<1, ID, OS_HI, OS_HI>(tmem, ah, bh, ACC ? k != 0 : true);
  }
}

// 8 values at a 16-byte chunk's hi and lo
__device__ __forceinline__ void os_store(unsigned char* p, const float* v) {
  uint4 h, l;
  split2(v[0], v[1], h.x, l.x);
  split2(v[2], v[3], h.y, l.y);
  split2(v[4], v[5], h.z, l.z);
  split2(v[6], v[7], h.w, l.w);
  *reinterpret_cast<uint4*>(p) = h;
  *reinterpret_cast<uint4*>(p + OS_PLANE) = l;
}
__device__ __forceinline__ void os_load(float (&x)[8], const unsigned char* p) {
  const uint4 h = *reinterpret_cast<const uint4*>(p), l = *reinterpret_cast<const uint4*>(p + OS_PLANE);
  const u32 hs[4] = {h.x, h.y, h.z, h.w}, ls[4] = {l.x, l.y, l.z, l.w};
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    float a, b, s, t;
    f16x2_float(hs[k], a, b);
    f16x2_float(ls[k], s, t);
    x[2 * k] = a + s;
    x[2 * k + 1] = b + t;
  }
}

}  // namespace tcb

extern "C" __global__ void __launch_bounds__(256, 1) tcb_orth_small(const tcb::Args a) {
  using namespace tcb;
  extern __shared__ unsigned char smem_raw[];
  __shared__ double sums[8];
  __shared__ __align__(8) u64 bar;
  __shared__ u32 tmem_slot;
  u32* err = reinterpret_cast<u32*>(a.p[15]);
  const u32 raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
  unsigned char* X = smem_raw + (base - raw);
  unsigned char* S = X + OS_XB * OS_BLOCK;
  unsigned char* P = S + OS_SB * OS_BLOCK;
  const u32 xa = base, sa = base + OS_XB * OS_BLOCK, pa = sa + OS_SB * OS_BLOCK, done = smem_u32(&bar);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    mbar_init(done, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" :: "r"(smem_u32(&tmem_slot)),
                 "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  for (u32 i = threadIdx.x; i < OS_XB * OS_BLOCK / 16; i += 256) reinterpret_cast<uint4*>(X)[i] = make_uint4(0, 0, 0, 0);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const u32 tmem = tmem_slot;
  grid_dependency_sync();
  if (blockIdx.x == 0 && threadIdx.x == 0 && err && (u64)a.p[15] == a.scratch) *err = 0u;

  const u32 m = (u32)a.p[0], n = (u32)a.p[1], count = m * n;
  const bool tall = m > n;
  const int steps = (int)a.p[2];
  const u32 s = tall ? n : m, len = tall ? m : n;
  const float* g = reinterpret_cast<const float*>(a.in[0]) + (u64)blockIdx.x * count;
  float* out = reinterpret_cast<float*>(a.out) + (u64)blockIdx.x * count;
  double sum = 0.0;
#pragma unroll 8
  for (u32 i = threadIdx.x; i < count; i += 256) {
    const double x = (double)ld1(g + i);
    sum += x * x;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) sums[warp] = sum;
  __syncthreads();
  sum = 0.0;
#pragma unroll
  for (int k = 0; k < 8; ++k) sum += sums[k];
  const double inv = 1.0 / (sqrt(sum) + (double)(TCB_NS_EPS)) * (double)(1u << TCB_EX);
#pragma unroll 4
  for (u32 i = threadIdx.x; i < count; i += 256) {
    const u32 row = i / n, col = i % n, r = tall ? col : row, c = tall ? row : col;
    u32 h, l;
    split2((float)((double)ld1(g + i) * inv), 0.0f, h, l);
    unsigned char* p = X + os_at(r, c) + 2 * (c & 7);
    *reinterpret_cast<unsigned short*>(p) = (unsigned short)h;
    *reinterpret_cast<unsigned short*>(p + OS_PLANE) = (unsigned short)l;
  }

  const u32 q = warp & 3, half = warp >> 2, row = 32 * q + lane;
  const u32 lanes = tmem + ((32 * q) << 16);
  const u32 long_steps = (len + 15) / 16, short_steps = (s + 15) / 16;
  u32 phase = 0;
  bool ok = true;
  // Everything written to shared memory is the tensor core's from here; the products run; their sums are ours.
  auto run = [&](auto issue) {
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    tc_fence_before();
    __syncthreads();
    if (warp == 0) {
      tc_fence_after();
      if (elect_one()) {
        issue();
        mma_commit(done);
      }
      __syncwarp();
    }
    ok = __syncthreads_and(mbar_wait(done, phase, nullptr, 1)) != 0;   // the same for every thread
    if (!ok && threadIdx.x == 0 && err) atomicCAS(err, 0u, 1u);
    phase ^= 1;
    tc_fence_after();
  };
  constexpr u32 W = TCB_ROWS / 2;   // columns of S and P a warp takes
  auto collect = [&](u32 c, float (&v)[32]) {
    float w[32], x[32];
    tmem_ld32(lanes + TCB_ROWS + c, w);
    tmem_ld32(lanes + 2 * TCB_ROWS + c, x);
    tmem_ld32(lanes + c, v);
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = __fadd_rn(v[i], __fadd_rn(w[i], x[i]));
  };
#pragma unroll 1
  for (int step = 0; step < steps && ok; ++step) {
    run([&] { os_product<TCB_ROWS, false, TCB_ROWS>(tmem, xa, xa, long_steps); });
#pragma unroll 1
    for (u32 c = half * W; c < (half + 1) * W; c += 32) {
      float v[32];
      collect(c, v);
      if (row < TCB_ROWS)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
#pragma unroll
          for (int i = 8 * k; i < 8 * k + 8; ++i) v[i] = row < s && c + i < s ? v[i] * pow2(TCB_ES - 2 * TCB_EX) : 0.0f;
          os_store(S + os_at(row, c + 8 * k), v + 8 * k);
        }
      __syncwarp();   // the accumulators are read by whole warps
    }
    run([&] { os_product<TCB_ROWS, false, TCB_ROWS>(tmem, sa, sa, short_steps); });
#pragma unroll 1
    for (u32 c = half * W; c < (half + 1) * W; c += 32) {
      float v[32];
      collect(c, v);
      if (row < TCB_ROWS)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          float x[8];
          os_load(x, S + os_at(row, c + 8 * k));
#pragma unroll
          for (int i = 0; i < 8; ++i)
            v[8 * k + i] = row < s && c + 8 * k + i < s
                               ? fmaf(TCB_NS_C, v[8 * k + i] * pow2(TCB_EP - 2 * TCB_ES), TCB_NS_B * (x[i] * pow2(TCB_EP - TCB_ES)))
                               : 0.0f;
          os_store(P + os_at(row, c + 8 * k), v + 8 * k);
        }
      __syncwarp();
    }
    run([&] {
      for (u32 b = 0; b * 64 < len; b += 4) {   // X in pieces of up to 256 columns
        const u32 at = xa + b * OS_BLOCK, left = len - b * 64;
        if (TCB_COLS >= 256 && left > 128) os_product<(TCB_COLS >= 256 ? 256 : 64), true, 0>(tmem + b * 64, pa, at, short_steps);
        else if (TCB_COLS >= 128 && left > 64) os_product<(TCB_COLS >= 128 ? 128 : 64), true, 0>(tmem + b * 64, pa, at, short_steps);
        else os_product<64, true, 0>(tmem + b * 64, pa, at, short_steps);
      }
    });
    const bool last = step == steps - 1;
#pragma unroll 1
    for (u32 c = 32 * half; c < len; c += 64) {
      float v[32];
      tmem_ld32(lanes + c, v);
      if (row < s)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        unsigned char* p = X + os_at(row, c + 8 * k);
        float x[8];
        os_load(x, p);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[8 * k + i] = fmaf(TCB_NS_A, x[i], v[8 * k + i] * pow2(-TCB_EP));
        if (!last) {
          os_store(p, v + 8 * k);   // columns beyond len: a zero's product is zero
        } else {
#pragma unroll
          for (int i = 8 * k; i < 8 * k + 8; ++i)
            if (c + i < len) out[tall ? (u64)(c + i) * n + row : (u64)row * n + c + i] = v[i] * pow2(-TCB_EX);
        }
      }
      __syncwarp();
    }
  }
  tc_fence_before();
  sync_settled(!ok);
  if (warp == 0) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" :: "r"(tmem), "r"(512u) : "memory");
  }
}
