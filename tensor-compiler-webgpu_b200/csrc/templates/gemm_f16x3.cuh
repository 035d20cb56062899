// tcb/gemm_f16x3.cuh -- a float32-accurate matrix product from fp16 tensor-core operands, with sizes
// known only at run time: the core of the operators whose operands this library splits itself
// (tcb/linear_nll.cuh, tcb/orthogonalize.cuh).
//
// An operand value x, scaled by a power of two s so that the largest one lies in [2^14, 2^15), is held
// as hi = fp16(x s) and lo = fp16(x s - hi): 22 significant bits, or an absolute error of 2^-25 where lo
// is subnormal, 2^-40 of the operand's largest value.  A product is
//   A.B ~= A_lo.B_hi + A_hi.B_lo + A_hi.B_hi     (A_lo.B_lo, below 2^-22 of a term, dropped)
// scaled back, exactly, in the epilogue.  The operands carry what the 3xTF32 split's do (tcb/gemm_tc.cuh:
// 11 + 11 bits too) at twice the rate and half the bytes: hi and lo together take the 4 bytes of the float
// they stand for.
//
// The tensor core truncates its float32 accumulator after every instruction, so a long chain drifts
// towards zero: by 3e-9 of the result a K index, measured (2.5e-5 at K = 8192).  A chain therefore ends
// after CHUNK indices; the epilogue warps add the chunks in registers, rounded to nearest, while the next
// one runs in the other TMEM accumulator.  With 256 the drift is below 1e-6; shorter chains leave the
// epilogue less time behind the products (K = 1024, exponentials in the epilogue: 10.8 ms with 256, 11.8
// with 128, 13.2 with 64).
//
// Persistent, one CTA per SM, warps specialised: warp 0 loads the stage's four tiles by TMA, one lane of
// warp 1 issues three tcgen05.mma.kind::f16 (M = 128, N = BN, K = 16) per K step into one of two TMEM
// accumulators, warps 4-11 collect the other: a quarter of the rows and half of the columns each, up to
// 128 sums a thread, on which the epilogue then runs 32 columns at a time.  They need more registers than
// an even share (168), so the first warpgroup gives up most of its own: 40 + 2 x 232 = 3 x 168.  Either operand may
// be K-major (64-byte rows) or MN-major (rows of 64 M or N values, 128 bytes), so no operand is ever
// transposed in memory.  A symmetric product (SYM) computes the tiles on or above the diagonal only and
// its epilogue mirrors them.
//
// p[0] = M, p[1] = N, p[2] = K, p[3] = batch, p[15] = error word; the rest is the epilogue's.
#pragma once
#include "tcb/sm100.cuh"

namespace tcb {

// two floats to packed fp16 (round to nearest even), a in the low half, and back
__device__ __forceinline__ u32 f16x2(float a, float b) {
  u32 r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  return r;
}
__device__ __forceinline__ void f16x2_float(u32 v, float& a, float& b) {
  asm("{\n .reg .b16 l, h;\n mov.b32 {l, h}, %2;\n cvt.f32.f16 %0, l;\n cvt.f32.f16 %1, h;\n}" : "=f"(a), "=f"(b) : "r"(v));
}
// hi and lo of two scaled values
__device__ __forceinline__ void split2(float a, float b, u32& hi, u32& lo) {
  hi = f16x2(a, b);
  float x, y;
  f16x2_float(hi, x, y);
  lo = f16x2(__fsub_rn(a, x), __fsub_rn(b, y));
}
// 2^k for k in [-126, 127]
__device__ __forceinline__ float pow2(int k) { return __uint_as_float((u32)(k + 127) << 23); }
// The exponent k of an operand's scale 2^k from its largest magnitude m (finite, >= 0): m 2^k in
// [2^14, 2^15).  Clamped so that 2^k and 2^-k are normal; a zero operand gives 0.
__device__ __forceinline__ int scale_exponent(float m) {
  if (!(m > 0.0f)) return 0;
  int e = (int)(__float_as_uint(m) >> 23) - 127;   // subnormal m: -127, so the scale stays below the bound
  e = 14 - e;
  return e > 126 ? 126 : e;
}

constexpr int HG_M = 128, HG_K = 32;
constexpr u32 HG_THREADS = 384;
template <int BN> struct F16x3 {
  static constexpr u32 A_BYTES = HG_M * HG_K * 2, B_BYTES = BN * HG_K * 2;
  static constexpr u32 STAGE = 2 * A_BYTES + 2 * B_BYTES;
  static constexpr u32 STAGING = 8 * 4096;                           // a 4 KB block per epilogue warp
  static constexpr u32 FIT = (227 * 1024 - 2048 - STAGING) / STAGE;  // 1 KB of barriers, 1 KB to align
  static constexpr u32 STAGES = FIT > 8 ? 8 : FIT;
};

// Shared-memory matrix descriptors.  K-major: 64-byte rows, 64-byte swizzle, 8-row groups 512 bytes
// apart.  MN-major: rows of 64 values along M or N, one per K index, 128-byte swizzle; 8-row groups 1 KB
// apart and the next 64 M or N values HG_K rows on.
__device__ __forceinline__ u64 f16_kdesc(u32 saddr) {
  return (u64)((saddr >> 4) & 0x3FFF) | (u64)1 << 16 | (u64)(512 >> 4) << 32 | (u64)1 << 46 | (u64)4 << 61;
}
__device__ __forceinline__ u64 f16_mndesc(u32 saddr) {
  return (u64)((saddr >> 4) & 0x3FFF) | (u64)((HG_K * 128) >> 4) << 16 | (u64)(1024 >> 4) << 32 | (u64)1 << 46 |
         (u64)2 << 61;
}
// D f32, A and B f16, M = 128, N = n
__host__ __device__ constexpr u32 idesc_f16(u32 n, u32 a_mn, u32 b_mn) {
  return (1u << 4) | (a_mn << 15) | (b_mn << 16) | ((n >> 3) << 17) | ((u32)(HG_M >> 4) << 24);
}
__device__ __forceinline__ void mma_f16(u32 tmem, u64 a, u64 b, u32 idesc, u32 accumulate) {
  asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
               " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}"
               :: "r"(tmem), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void tmem_ld32(u32 taddr, float (&r)[32]) {
  u32 v[32];
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
               "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
                 "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]),
                 "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]),
                 "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
               : "r"(taddr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int j = 0; j < 32; ++j) r[j] = __uint_as_float(v[j]);
}

struct F16Tile { int m0, n0, bz; u32 mt, nt; };

// Unit u -> output tile.  Grouped raster (8 tile rows per group) so the CTAs running together share
// operand panels in L2; a symmetric product walks the tiles that reach the diagonal, row by row.
template <int BN, bool SYM>
__device__ __forceinline__ F16Tile f16_tile(u32 u, u32 tm, u32 tn, u32 per) {
  F16Tile T;
  T.bz = (int)(u / per);
  u32 r = u % per;
  if (SYM) {
    u32 i = 0;
    for (;; ++i) {
      const u32 first = i * HG_M / BN, n = tn - first;
      if (r < n) { T.nt = first + r; break; }
      r -= n;
    }
    T.mt = i;
  } else {
    const u32 g = r / (8 * tn), first = g * 8;
    const u32 gsz = tm - first < 8 ? tm - first : 8;
    const u32 w = r - first * tn;
    T.mt = first + w % gsz;
    T.nt = w / gsz;
  }
  T.m0 = (int)(T.mt * HG_M);
  T.n0 = (int)(T.nt * BN);
  return T;
}
template <int BN, bool SYM>
__device__ __forceinline__ u32 f16_units(u32 tm, u32 tn) {
  if (!SYM) return tm * tn;
  u32 n = 0;
  for (u32 i = 0; i < tm; ++i) n += tn - i * HG_M / BN;
  return n;
}

// An epilogue warp's view of one tile: rows 32 q .. of it, columns from c0, this lane's row.
struct F16Epi {
  F16Tile T;
  int q, c0, lane;
  u64 row;             // of the output, may lie beyond M
  u32 stage;           // shared-memory address of the warp's 4 KB block
  unsigned char* gstage;
};

// Written out block by block, so that every index into the sums is a constant and they stay in registers.
template <int I, int NB>
__device__ __forceinline__ void f16_collect(float (&v)[NB][32], u32 t) {
  if constexpr (I < NB) {
    float w[32];
    tmem_ld32(t + 32 * I, w);
#pragma unroll
    for (int i = 0; i < 32; ++i) v[I][i] = __fadd_rn(v[I][i], w[i]);
    f16_collect<I + 1>(v, t);
  }
}
template <int I, int NB, class EPI>
__device__ __forceinline__ void f16_blocks(EPI& epi, const F16Epi& e, float (&v)[NB][32], u32 N) {
  if constexpr (I < NB) {
    if ((u32)(e.T.n0 + e.c0 + 32 * I) < N) epi.block(e, e.c0 + 32 * I, v[I]);
    f16_blocks<I + 1>(epi, e, v, N);
  }
}

// EPI: struct with begin(e), block(e, c0, v) for each 32 columns (from column c0 of the tile) that reach into
// the output, end(e), and done(e) once after the last tile.
template <int BN, bool A_MN, bool B_MN, bool SYM, int CHUNK, class EPI>
__device__ __forceinline__ void gemm_f16x3(const GemmParams& P, EPI& epi) {
  using S = F16x3<BN>;
  constexpr int STAGES = (int)S::STAGES;
  extern __shared__ unsigned char smem_raw[];
  u32* err = reinterpret_cast<u32*>(P.a.p[15]);
  const u32 raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
  unsigned char* gbase = smem_raw + (base - raw);
  const u32 bars = base + STAGES * S::STAGE, staging = bars + 1024;
  u32* tmem_slot = reinterpret_cast<u32*>(gbase + STAGES * S::STAGE + (2 * STAGES + 4) * 8);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  auto full = [&](int s) { return bars + 8u * s; };
  auto empty = [&](int s) { return bars + 8u * (STAGES + s); };
  auto accf = [&](u32 b) { return bars + 8u * (2 * STAGES + b); };
  auto acce = [&](u32 b) { return bars + 8u * (2 * STAGES + 2 + b); };
  const u32 M = (u32)P.a.p[0], N = (u32)P.a.p[1], K = (u32)P.a.p[2], batch = (u32)P.a.p[3];
  const u32 tm = (M + HG_M - 1) / HG_M, tn = (N + BN - 1) / BN, kbs = (K + HG_K - 1) / HG_K;
  const u32 per = f16_units<BN, SYM>(tm, tn), units = per * batch;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) { mbar_init(full(s), 1); mbar_init(empty(s), 1); }
    for (u32 b = 0; b < 2; ++b) { mbar_init(accf(b), 1); mbar_init(acce(b), 8); }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" :: "r"(smem_u32(tmem_slot)),
                 "r"((u32)(2 * BN)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const u32 tmem = *tmem_slot;
  grid_dependency_sync();   // the set-up above touched this CTA's shared and tensor memory only

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
    if (warp == 0 && lane == 0) {
      u32 it = 0;
      bool ok = true;
      for (u32 u = blockIdx.x; ok && u < units; u += gridDim.x) {
        const F16Tile T = f16_tile<BN, SYM>(u, tm, tn, per);
        for (u32 kb = 0; kb < kbs; ++kb, ++it) {
          const int s = it % STAGES;
          if (it >= (u32)STAGES && !mbar_wait(empty(s), ((it / STAGES) - 1) & 1, err, 1)) { ok = false; break; }
          const u32 st = base + s * S::STAGE;
          const int kc = (int)(kb * HG_K);
          mbar_expect_tx(full(s), S::STAGE);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const u32 a = st + h * S::A_BYTES, b = st + 2 * S::A_BYTES + h * S::B_BYTES;
            if (A_MN) {
#pragma unroll
              for (int c = 0; c < HG_M / 64; ++c) tma_load_3d(a + c * HG_K * 128, &P.maps[h], full(s), T.m0 + 64 * c, kc, T.bz);
            } else {
              tma_load_3d(a, &P.maps[h], full(s), kc, T.m0, T.bz);
            }
            if (B_MN) {
#pragma unroll
              for (int c = 0; c < BN / 64; ++c) tma_load_3d(b + c * HG_K * 128, &P.maps[2 + h], full(s), T.n0 + 64 * c, kc, T.bz);
            } else {
              tma_load_3d(b, &P.maps[2 + h], full(s), kc, T.n0, T.bz);
            }
          }
        }
      }
      // wait (bounded) for the copies still in flight before this CTA may exit
      for (u32 i = it > (u32)STAGES ? it - STAGES : 0; i < it; ++i) mbar_wait(full(i % STAGES), (i / STAGES) & 1, err, 2);
    } else if (warp == 1 && lane == 0) {
      constexpr u32 ID = idesc_f16(BN, A_MN ? 1u : 0u, B_MN ? 1u : 0u);
      auto da = [&](u32 t, int k) { return A_MN ? f16_mndesc(t + 2048 * k) : f16_kdesc(t + 32 * k); };
      auto db = [&](u32 t, int k) { return B_MN ? f16_mndesc(t + 2048 * k) : f16_kdesc(t + 32 * k); };
      u32 it = 0, j = 0;   // stages, chunks
      bool ok = true;
      for (u32 u = blockIdx.x; ok && u < units; u += gridDim.x) {
        for (u32 k0 = 0; ok && k0 < kbs; k0 += CHUNK / HG_K, ++j) {
          const u32 k1 = k0 + CHUNK / HG_K < kbs ? k0 + CHUNK / HG_K : kbs, buf = j & 1;
          if (j >= 2 && !mbar_wait(acce(buf), ((j >> 1) - 1) & 1, err, 5)) { ok = false; break; }
          tc_fence_after();
          const u32 acc = tmem + buf * BN;
          for (u32 kb = k0; kb < k1; ++kb, ++it) {
            const int s = it % STAGES;
            if (!mbar_wait(full(s), (it / STAGES) & 1, err, 3)) { ok = false; break; }
            tc_fence_after();
            const u32 st = base + s * S::STAGE;
#pragma unroll
            for (int k = 0; k < HG_K / 16; ++k) {
              const u64 ah = da(st, k), al = da(st + S::A_BYTES, k);
              const u64 bh = db(st + 2 * S::A_BYTES, k), bl = db(st + 2 * S::A_BYTES + S::B_BYTES, k);
              mma_f16(acc, al, bh, ID, ((kb - k0) | k) != 0);
              mma_f16(acc, ah, bl, ID, 1);
              mma_f16(acc, ah, bh, ID, 1);
            }
            mma_commit(empty(s));
          }
          if (ok) mma_commit(accf(buf));
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 232;");
    constexpr int NB = BN / 64;   // 32-column blocks a warp
    F16Epi e;
    e.q = warp & 3;
    e.c0 = (warp - 4) / 4 * (BN / 2);
    e.lane = lane;
    e.stage = staging + (u32)(warp - 4) * 4096;
    e.gstage = gbase + (e.stage - base);
    u32 j = 0;
    bool ok = true;
    for (u32 u = blockIdx.x; ok && u < units; u += gridDim.x) {
      e.T = f16_tile<BN, SYM>(u, tm, tn, per);
      e.row = (u64)e.T.m0 + 32 * e.q + lane;
      float v[NB][32];
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int i = 0; i < 32; ++i) v[b][i] = 0.0f;
      for (u32 k0 = 0; k0 < kbs; k0 += CHUNK / HG_K, ++j) {
        const u32 buf = j & 1;
        if (!mbar_wait(accf(buf), (j >> 1) & 1, err, 4)) { ok = false; break; }
        tc_fence_after();
        const u32 t = tmem + buf * BN + ((u32)(32 * e.q) << 16) + (u32)e.c0;
        f16_collect<0>(v, t);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" :: "r"(acce(buf)) : "memory");
      }
      // this warp's part of the tile reaches into the output
      if (ok && (u32)e.T.m0 + 32 * e.q < M && (u32)(e.T.n0 + e.c0) < N) {
        epi.begin(e);
        f16_blocks<0>(epi, e, v, N);
        epi.end(e);
      }
    }
    epi.done(e);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" :: "r"(tmem), "r"((u32)(2 * BN)) : "memory");
  }
}

// ---- what epilogues share ----

// 32 columns of hi / lo pairs through the warp's staging block to two planes of an fp16 array by TMA
// store (map 4: {cols, rows, planes}, boxes of 32 x 32, 64-byte swizzle).
__device__ __forceinline__ void store_split32(const F16Epi& e, const TmaDesc* map, const float (&v)[32], int col,
                                              int row, int plane_hi, int plane_lo) {
  if (e.lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");   // the last store has read it
  __syncwarp();
  uint4* sp = reinterpret_cast<uint4*>(e.gstage);
  const int sw = (e.lane >> 1) & 3;
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    uint4 h, l;
    split2(v[8 * c], v[8 * c + 1], h.x, l.x);
    split2(v[8 * c + 2], v[8 * c + 3], h.y, l.y);
    split2(v[8 * c + 4], v[8 * c + 5], h.z, l.z);
    split2(v[8 * c + 6], v[8 * c + 7], h.w, l.w);
    sp[e.lane * 4 + (c ^ sw)] = h;
    sp[128 + e.lane * 4 + (c ^ sw)] = l;
  }
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  __syncwarp();
  if (e.lane == 0) {
    tma_store_3d(map, e.stage, col, row, plane_hi);
    tma_store_3d(map, e.stage + 2048, col, row, plane_lo);
    bulk_commit();
  }
}

// 32 x 32 floats, a row per lane, turned in the warp's staging block so that lane l holds column l
// of row r in v[r]: rows are then written (or added to) 32 consecutive floats at a time, whatever the
// output's row stride.
__device__ __forceinline__ void turn32(const F16Epi& e, float (&v)[32]) {
  float4* sp = reinterpret_cast<float4*>(e.gstage);
  __syncwarp();
#pragma unroll
  for (int c = 0; c < 8; ++c)
    sp[e.lane * 8 + (c ^ (e.lane & 7))] = make_float4(v[4 * c], v[4 * c + 1], v[4 * c + 2], v[4 * c + 3]);
  __syncwarp();
  const float* sf = reinterpret_cast<const float*>(sp);
#pragma unroll
  for (int r = 0; r < 32; ++r) v[r] = sf[r * 32 + (((e.lane >> 2) ^ (r & 7)) << 2) + (e.lane & 3)];
}

// Sums over the warp's 32 rows of 32 columns: lane l gets column l's.  Halves are exchanged, so the
// additions are 31 a lane, in a fixed order.
__device__ __forceinline__ float column_sums32(float (&v)[32], int lane) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const bool up = (lane & o) != 0;
#pragma unroll
    for (int j = 0; j < o; ++j) {
      const float send = up ? v[j] : v[j + o], keep = up ? v[j + o] : v[j];
      v[j] = __fadd_rn(keep, __shfl_xor_sync(0xffffffffu, send, o));
    }
  }
  return v[0];
}

}  // namespace tcb
