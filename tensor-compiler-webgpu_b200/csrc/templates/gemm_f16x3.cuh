// tcb/gemm_f16x3.cuh -- a float32-accurate matrix product from fp16 tensor-core operands, with sizes
// known only at run time: the core of the operators whose operands this library splits itself
// (tcb/linear_nll.cuh, tcb/orthogonalize.cuh).
//
// An operand value x, scaled by a power of two s so that the largest one lies in [2^14, 2^15), is held
// as hi = fp16(x s) and lo = fp16(x s - hi): 22 significant bits, or an absolute error of 2^-25 where lo
// is subnormal, up to 2^-39 of the operand's largest value.  A product is
//   A.B ~= A_lo.B_hi + A_hi.B_lo + A_hi.B_hi     (A_lo.B_lo, below 2^-22 of a term, dropped)
// scaled back, exactly, in the epilogue.  The operands carry what the 3xTF32 split's do (tcb/gemm_tc.cuh:
// 11 + 11 bits too) at twice the rate and half the bytes: hi and lo together take the 4 bytes of the float
// they stand for.
//
// The tensor core truncates its float32 accumulator after every instruction, so a long chain drifts
// towards zero: by 3e-9 of the result a K index, measured (2.5e-5 at K = 8192).  A chain therefore ends
// after CHUNK indices; the epilogue warps add the chunks in registers, rounded to nearest, while the next
// one runs in the other TMEM buffer.  With 256 the drift is below 1e-6; shorter chains leave the epilogue
// less time behind the products (K = 1024, exponentials in the epilogue: 10.8 ms with 256, 11.8 with 128,
// 13.2 with 64).  Tiles narrower than 256 have TMEM to spare: their mixed terms go to accumulators of
// their own, which keeps the drift of the main one to a third and breaks up the chain of dependent
// instructions (a 64-wide product takes about 100 clocks in a chain, 32 by its size).
//
// Persistent, one CTA per SM, warps specialised: warp 0 loads the stage's four tiles by TMA, one lane of
// warp 1 issues three tcgen05.mma.kind::f16 (M = 128 or, for a pair, 256, N = BN, K = 16) per K step into one of
// two TMEM buffers, warps 4-11 collect the other: a quarter of the rows and half of the columns each, up to 128
// sums a thread, on which the epilogue then runs 32 columns at a time.  They need more registers than an
// even share (168), so the first warpgroup gives up most of its own: 40 + 2 x 232 = 3 x 168.  Either
// operand may be K-major (64-byte rows) or MN-major (rows of 64 M or N values, 128 bytes), so no operand is
// ever transposed in memory.  A symmetric product (SYM) computes the tiles on or above the diagonal only
// and its epilogue mirrors them.
//
// Pairs (CTAS = 2): two SMs work on a tile of 256 rows, each loading 128 rows of A and half of B's columns, and
// the even one's warp 1 issues the products of both (cta_group::2).  A stage of 32 K indices of a tile 256 wide
// takes 768 clocks of products; one SM alone would load 48 KB in them, as many bytes a clock as it takes from L2
// at best (64, measured with boxes of 16 KB), one of a pair 32 KB: 16384 x 1024 x 131072 with exponentials 10.9
// ms alone, 9.2 in pairs.  A K step of 16 takes 290 to 310 ns in long products, the epilogues' share included
// (1.5 to 1.6 PFLOP/s of products), 320 to 380 when run for seconds.  128 wide a pair is as fast as two SMs (164 to
// 200 ns a step), but draws less power: 4095 x 256 x 8192 forward and backward, run for seconds, 269 us alone and 261
// in pairs.  Full barriers are the even CTA's and count both CTAs' bytes,
// empty and accumulator ones are each CTA's own, and both leave together.
//
// Work: where there are as many tiles as SMs or more, they go whole to the CTAs in turn, in grouped raster
// order (full = tiles).  Fewer ones may be divided (full = 0): they are one line of units of `quantum` chunks,
// cut into equal runs, one a CTA.  A run that holds a part of a tile only leaves its sums in scratch; the warp
// that arrives last at its part of the tile adds them all, in order, and goes on to the epilogue: no CTA waits
// for another, and the result does not depend on which came last.
//
// p[0] = M | N << 32, p[1] = K | batch << 32, p[2] = full | quantum << 32, p[3] = byte offset in scratch of
// the partial sums (two 128 x BN slots a CTA), p[15] = control block: the error word, 16 bytes on a
// counter per warp and divided tile (fewer than 148 tiles), zero between launches.  Maps: A, B ({cols, rows,
// 2 batch}: each matrix's hi plane, then its lo plane, a box taking both) and the epilogue's.  A kernel may run
// two products side by side, each on CTAs of its own (F16Job).  BLOCKED operands (no batch) are stored in
// blocks of 256 columns, a block's planes of 512-byte rows in the place of a batch: with rows as long as a
// vocabulary every row of a K-major box lies in a page of its own (dh at 8192 x 1024 x 50001: 1.34 us a stage
// of 32 K indices, the same product of short rows 0.70).
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
// Two float32 operations in one instruction, each rounded to nearest: the epilogues' warps, two an SM
// quarter, wait on what they issue (dz at 4095 x 256 x 8192: 73.2 us with single operations and every column
// compared with the target, 70.0 so).
__device__ __forceinline__ u64 pair2(float a, float b) {
  u64 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpair2(u64 r, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(r)); }
__device__ __forceinline__ void add2(float& a, float& b, float x, float y) {
  u64 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(pair2(a, b)), "l"(pair2(x, y)));
  unpair2(r, a, b);
}
__device__ __forceinline__ void mul2(float& a, float& b, float x, float y) {
  u64 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(pair2(a, b)), "l"(pair2(x, y)));
  unpair2(r, a, b);
}
// a = a x + c, b = b y + d
__device__ __forceinline__ void fma2(float& a, float& b, float x, float y, float c, float d) {
  u64 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(pair2(a, b)), "l"(pair2(x, y)), "l"(pair2(c, d)));
  unpair2(r, a, b);
}
template <int N> __device__ __forceinline__ void add32(float (&v)[N], const float (&w)[N]) {
#pragma unroll
  for (int i = 0; i < N; i += 2) add2(v[i], v[i + 1], w[i], w[i + 1]);
}
// hi and lo of two scaled values
__device__ __forceinline__ void split2(float a, float b, u32& hi, u32& lo) {
  hi = f16x2(a, b);
  float x, y;
  f16x2_float(hi, x, y);
  fma2(x, y, -1.0f, -1.0f, a, b);
  lo = f16x2(x, y);
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
constexpr int f16_accs(int bn) { return bn == 256 ? 1 : bn == 128 ? 2 : 3; }   // accumulators of a TMEM buffer
template <int BN, int CTAS> struct F16x3 {
  static constexpr int TM = CTAS * HG_M, COLS = BN / CTAS;   // tile rows; columns of B a CTA loads
  static constexpr u32 A_BYTES = HG_M * HG_K * 2, B_BYTES = COLS * HG_K * 2;
  static constexpr u32 STAGE = 2 * A_BYTES + 2 * B_BYTES;
  static constexpr u32 BARS = 256, VECTORS = 8 * 128, STAGING = 8 * 4096;   // 128 bytes, a 4 KB block an epilogue warp
  static constexpr u32 FIT = (227 * 1024 - 1024 - BARS - VECTORS - STAGING) / STAGE;   // 1 KB to align the ring
  static constexpr u32 STAGES = FIT > 8 ? 8 : FIT;
  static constexpr u32 ACCS = f16_accs(BN);
  static constexpr u32 TMEM = 512;                                   // columns allocated: 2 ACCS BN, a power of 2
};

// Shared-memory matrix descriptors.  K-major: 64-byte rows, 64-byte swizzle, 8-row groups 512 bytes
// apart.  MN-major: rows of 64 values along M or N, one per K index, 128-byte swizzle; 8-row groups 1 KB
// apart and the next 64 M or N values 2 HG_K rows on (their lo plane lies between).  Only the address in the
// low word changes.
template <bool MN> __device__ __forceinline__ u32 f16_desc_lo(u32 saddr) {
  return (saddr >> 4) | (MN ? (2 * HG_K * 128) >> 4 : 1) << 16;
}
template <bool MN> __host__ __device__ constexpr u32 f16_desc_hi() {
  return MN ? 1024u >> 4 | 1u << 14 | 2u << 29 : 512u >> 4 | 1u << 14 | 4u << 29;
}
// D f32, A and B f16
__host__ __device__ constexpr u32 idesc_f16(u32 m, u32 n, u32 a_mn, u32 b_mn) {
  return (1u << 4) | (a_mn << 15) | (b_mn << 16) | ((n >> 3) << 17) | ((m >> 4) << 24);
}
__device__ __forceinline__ bool elect_one() {
  u32 p;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(p));
  return p != 0;
}
template <int CTAS, u32 ID, u32 AH, u32 BH>
__device__ __forceinline__ void mma_f16(u32 tmem, u32 a, u32 b, bool accumulate) {
  if constexpr (CTAS == 2)
    asm volatile("{\n .reg .pred p;\n .reg .b64 x, y;\n setp.ne.b32 p, %3, 0;\n mov.b64 x, {%1, %5};\n mov.b64 y, {%2, %6};\n"
                 " tcgen05.mma.cta_group::2.kind::f16 [%0], x, y, %4, p;\n}"
                 :: "r"(tmem), "r"(a), "r"(b), "r"((u32)accumulate), "n"(ID), "n"(AH), "n"(BH) : "memory");
  else
    asm volatile("{\n .reg .pred p;\n .reg .b64 x, y;\n setp.ne.b32 p, %3, 0;\n mov.b64 x, {%1, %5};\n mov.b64 y, {%2, %6};\n"
                 " tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %4, p;\n}"
                 :: "r"(tmem), "r"(a), "r"(b), "r"((u32)accumulate), "n"(ID), "n"(AH), "n"(BH) : "memory");
}

// ---- a pair of CTAs (a cluster of two, the even one its leader) ----
__device__ __forceinline__ u32 pair_rank() { u32 r; asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ void pair_sync() {
  asm volatile("barrier.cluster.arrive.release;\n barrier.cluster.wait.acquire;" ::: "memory");
}
// this CTA's shared-memory address in the leader
__device__ __forceinline__ u32 in_leader(u32 addr) {
  u32 r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(addr));
  return r;
}
// a tile into this CTA, its bytes counted by a barrier of the pair's
__device__ __forceinline__ void pair_load_3d(u32 dst, const TmaDesc* map, u32 bar, int c0, int c1, int c2) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 "
               "[%0], [%1, {%2, %3, %4}], [%5];"
               :: "r"(dst), "l"(reinterpret_cast<u64>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(bar) : "memory");
}
// arrives at the same barrier of both CTAs when the pair's products so far are done
__device__ __forceinline__ void pair_commit(u32 bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
               :: "r"(bar), "h"((unsigned short)3) : "memory");
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

struct F16Tile { int m0, n0, bz; };

// Tile u.  Grouped raster (8 tile rows per group) so the CTAs running together share operand panels in L2;
// a symmetric product walks the tiles that reach the diagonal, row by row.
template <int BN, int CTAS, bool SYM>
__device__ __forceinline__ F16Tile f16_tile(u32 u, u32 tm, u32 tn, u32 per) {
  F16Tile T;
  T.bz = (int)(u / per);
  u32 r = u % per, mt, nt;
  if (SYM) {
    u32 i = 0;
    for (;; ++i) {
      const u32 first = i * CTAS * HG_M / BN, n = tn - first;
      if (r < n) { nt = first + r; break; }
      r -= n;
    }
    mt = i;
  } else {
    const u32 g = r / (8 * tn), first = g * 8;
    const u32 gsz = tm - first < 8 ? tm - first : 8;
    const u32 w = r - first * tn;
    mt = first + w % gsz;
    nt = w / gsz;
  }
  T.m0 = (int)(mt * CTAS * HG_M);
  T.n0 = (int)(nt * BN);
  return T;
}
template <int BN, int CTAS, bool SYM>
__device__ __forceinline__ u32 f16_tiles(u32 tm, u32 tn) {
  if (!SYM) return tm * tn;
  u32 n = 0;
  for (u32 i = 0; i < tm; ++i) n += tn - i * CTAS * HG_M / BN;
  return n;
}

// The work of one CTA or pair, in order: whole tiles, then its run of the divided ones.
struct F16Work {
  u32 tiles, full, chunks, quantum, per;   // per: units of a divided tile
  u32 grid, u;                             // CTAs (or pairs); next whole tile
  u64 at, end, total;                      // the run, in units over the divided tiles
  u32 tile, c0, c1;                        // the current piece: chunks c0 .. c1 of a tile
  __device__ __forceinline__ F16Work(u32 tiles_, u32 full_, u32 chunks_, u32 quantum_, u32 block, u32 grid_)
      : tiles(tiles_), full(full_), chunks(chunks_), quantum(quantum_), per((chunks_ + quantum_ - 1) / quantum_),
        grid(grid_), u(block) {
    total = (u64)(tiles - full) * per;
    at = block * total / grid;
    end = (block + 1) * total / grid;
  }
  __device__ __forceinline__ bool next() {
    if (u < full) {
      tile = u;
      c0 = 0;
      c1 = chunks;
      u += grid;
      return true;
    }
    if (at >= end) return false;
    const u32 t = (u32)(at / per), k = (u32)(at - (u64)t * per);
    const u32 n = (u32)(end - at < per - k ? end - at : per - k);
    tile = full + t;
    c0 = k * quantum;
    c1 = (k + n) * quantum < chunks ? (k + n) * quantum : chunks;
    at += n;
    return true;
  }
  __device__ __forceinline__ bool whole() const { return c0 == 0 && c1 == chunks; }
  // the CTA whose run holds unit x
  __device__ __forceinline__ u32 owner(u64 x) const { return (u32)(((x + 1) * grid - 1) / total); }
};

// An epilogue warp's view of one tile: rows 32 q .. of it, columns from c0, this lane's row.
struct F16Epi {
  F16Tile T;
  int q, c0, lane;
  u64 row;             // of the output, may lie beyond M
  u32 M, N;
  u32 stage;           // shared-memory address of the warp's 4 KB block
  unsigned char* gstage;
  float* vec;          // 32 floats of the warp's own
};

// Written out block by block, so that every index into the sums is a constant and they stay in registers.
template <int BN, int I, int NB>
__device__ __forceinline__ void f16_collect(float (&v)[NB][32], u32 t) {
  if constexpr (I < NB) {
    constexpr int ACCS = f16_accs(BN);
    float w[32];
    if constexpr (ACCS > 1) {   // the mixed terms, 2^-11 of the main ones, first
      tmem_ld32(t + BN + 32 * I, w);
      if constexpr (ACCS > 2) {
        float x[32];
        tmem_ld32(t + 2 * BN + 32 * I, x);
        add32(w, x);
      }
      float x[32];
      tmem_ld32(t + 32 * I, x);
      add32(w, x);
    } else {
      tmem_ld32(t + 32 * I, w);
    }
    add32(v[I], w);
    f16_collect<BN, I + 1>(v, t);
  }
}
// A warp's sums to or from a partial slot: 32 lanes side by side, 64 loads in flight.
template <bool ADD, int NB>
__device__ __forceinline__ void f16_partial_load(float (&v)[NB][32], const float* p) {
  constexpr int STEP = NB > 1 ? 2 : 1;
#pragma unroll
  for (int b = 0; b < NB; b += STEP) {
    float w[STEP][32];
#pragma unroll
    for (int k = 0; k < STEP; ++k)
#pragma unroll
      for (int i = 0; i < 32; ++i) w[k][i] = __ldcg(p + ((b + k) * 32 + i) * 32);
#pragma unroll
    for (int k = 0; k < STEP; ++k)
#pragma unroll
      for (int i = 0; i < 32; ++i) v[b + k][i] = ADD ? __fadd_rn(v[b + k][i], w[k][i]) : w[k][i];
  }
}
template <int I, int NB>
__device__ __forceinline__ void f16_partial_store(const float (&v)[NB][32], float* p) {
  if constexpr (I < NB) {
#pragma unroll
    for (int i = 0; i < 32; ++i) __stcg(p + (I * 32 + i) * 32, v[I][i]);
    f16_partial_store<I + 1>(v, p);
  }
}
template <int I, int NB, class EPI>
__device__ __forceinline__ void f16_blocks(EPI& epi, const F16Epi& e, float (&v)[NB][32], u32 N) {
  if constexpr (I < NB) {
    if ((u32)(e.T.n0 + e.c0 + 32 * I) < N) epi.block(e, e.c0 + 32 * I, v[I]);
    f16_blocks<I + 1>(epi, e, v, N);
  }
}

// EPI: struct with start(staging) once, by all 256 epilogue threads, begin(e) before a tile's or part's products
// have come, block(e, c0, v) for each 32 columns (from column c0 of the tile) that reach into the output, end(e),
// and done(e) once after the last tile.
struct F16Job {
  const TmaDesc *ma, *mb;
  u32 M, N, K, batch, full, quantum, block, grid;
  float* part;
  u32* counters;
};
__device__ __forceinline__ F16Job f16_job(const GemmParams& P) {
  return {&P.maps[0], &P.maps[1], (u32)P.a.p[0], (u32)((u64)P.a.p[0] >> 32), (u32)P.a.p[1], (u32)((u64)P.a.p[1] >> 32),
          (u32)P.a.p[2], (u32)((u64)P.a.p[2] >> 32), blockIdx.x, gridDim.x,
          reinterpret_cast<float*>(P.a.scratch + (u64)P.a.p[3]), reinterpret_cast<u32*>(P.a.p[15]) + 4};
}

template <int BN, int CTAS, bool A_MN, bool B_MN, bool SYM, bool BLOCKED, int CHUNK, class EPI>
__device__ __forceinline__ void gemm_f16x3(const F16Job& J, u32* err, EPI& epi) {
  using S = F16x3<BN, CTAS>;
  constexpr u32 STAGES = S::STAGES;
  extern __shared__ unsigned char smem_raw[];
  const u32 raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
  unsigned char* gbase = smem_raw + (base - raw);
  const u32 staging = base + STAGES * S::STAGE, bars = staging + S::STAGING, vectors = bars + S::BARS;
  u32* tmem_slot = reinterpret_cast<u32*>(gbase + (bars - base) + (2 * STAGES + 4) * 8);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  auto full = [&](u32 s) { return bars + 8u * s; };
  auto empty = [&](u32 s) { return bars + 8u * (STAGES + s); };
  auto accf = [&](u32 b) { return bars + 8u * (2 * STAGES + b); };
  auto acce = [&](u32 b) { return bars + 8u * (2 * STAGES + 2 + b); };
  const u32 M = J.M, N = J.N;
  constexpr u32 TM = S::TM;
  const u32 rank = CTAS == 2 ? pair_rank() : 0, unit = J.block / CTAS;   // a CTA, or a pair
  const u32 tm = (M + TM - 1) / TM, tn = (N + BN - 1) / BN, kbs = (J.K + HG_K - 1) / HG_K;
  constexpr u32 CK = CHUNK / HG_K;   // stages of a chunk
  const u32 per = f16_tiles<BN, CTAS, SYM>(tm, tn);
  F16Work work(per * J.batch, J.full, (kbs + CK - 1) / CK, J.quantum, unit, J.grid / CTAS);

  if (threadIdx.x == 32 * 3) {
    asm volatile("prefetch.tensormap [%0];" :: "l"(reinterpret_cast<u64>(J.ma)) : "memory");
    asm volatile("prefetch.tensormap [%0];" :: "l"(reinterpret_cast<u64>(J.mb)) : "memory");
  }
  if (threadIdx.x == 0) {
    for (u32 s = 0; s < STAGES; ++s) { mbar_init(full(s), 1); mbar_init(empty(s), 1); }
    for (u32 b = 0; b < 2; ++b) { mbar_init(accf(b), 1); mbar_init(acce(b), 8 * CTAS); }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    if constexpr (CTAS == 2) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" :: "r"(smem_u32(tmem_slot)),
                   "r"(S::TMEM) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" :: "r"(smem_u32(tmem_slot)),
                   "r"(S::TMEM) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (CTAS == 2) pair_sync();   // both CTAs' barriers are set up
  tc_fence_after();
  const u32 tmem = *tmem_slot;
  grid_dependency_sync();   // the set-up above touched this CTA's shared and tensor memory only

  bool ok = true;   // this thread's waits have not given up
  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
    // Both warps run their loops whole and one elected lane issues: the operands of the copies and products are
    // then the warp's, held in uniform registers.  Issued from a one-lane branch each product cost some 120
    // clocks to issue, whatever its size; a wait's outcome is voted on so that the branches stay uniform too.
    const bool leader = elect_one();
    auto wait = [&](u32 bar, u32 parity, u32 code) { return __all_sync(0xffffffffu, mbar_wait(bar, parity, err, code)) != 0; };
    if (warp == 0) {
      u32 it = 0, s = 0, phase = 0;
      while (ok && work.next()) {
        const F16Tile T = f16_tile<BN, CTAS, SYM>(work.tile, tm, tn, per);
        const u32 kend = work.c1 * CK < kbs ? work.c1 * CK : kbs;
        for (u32 kb = work.c0 * CK; kb < kend; ++kb, ++it) {
          if (it >= STAGES && !wait(empty(s), phase ^ 1, 1)) { ok = false; break; }
          const u32 st = base + s * S::STAGE, sb = st + 2 * S::A_BYTES;
          const int kc = (int)(kb * HG_K);
          const u32 bar = CTAS == 2 ? in_leader(full(s)) : full(s);
          const int m0 = T.m0 + (int)rank * HG_M, n0 = T.n0 + (int)rank * S::COLS;
          auto load = [&](u32 dst, const TmaDesc* map, int col, int row) {
            const int c = BLOCKED ? col & 255 : col, z = BLOCKED ? 2 * (col >> 8) : 2 * T.bz;
            if constexpr (CTAS == 2) pair_load_3d(dst, map, bar, c, row, z);
            else tma_load_3d(dst, map, bar, c, row, z);
          };
          if (leader) {
            if (rank == 0) mbar_expect_tx(full(s), CTAS * S::STAGE);
            // a box holds a tile's hi plane and, behind it, its lo plane
            if (A_MN) {
#pragma unroll
              for (int c = 0; c < HG_M / 64; ++c) load(st + c * HG_K * 256, J.ma, m0 + 64 * c, kc);
            } else {
              load(st, J.ma, kc, m0);
            }
            if (B_MN) {
#pragma unroll
              for (int c = 0; c < S::COLS / 64; ++c) load(sb + c * HG_K * 256, J.mb, n0 + 64 * c, kc);
            } else {
              load(sb, J.mb, kc, n0);
            }
          }
          __syncwarp();
          if (++s == STAGES) { s = 0; phase ^= 1; }
        }
      }
      // wait (bounded) for the copies still in flight before this CTA (the leader: the pair) may exit
      if (rank == 0) for (u32 i = it > STAGES ? it - STAGES : 0; i < it; ++i) ok &= mbar_wait(full(i % STAGES), (i / STAGES) & 1, err, 2);
    } else if (warp == 1 && rank == 0) {
      constexpr u32 ID = idesc_f16(TM, BN, A_MN ? 1u : 0u, B_MN ? 1u : 0u), AH = f16_desc_hi<A_MN>(), BH = f16_desc_hi<B_MN>();
      // hi to lo plane, and one K step on, in descriptor units of 16 bytes
      constexpr u32 AL = (A_MN ? HG_K * 128 : S::A_BYTES) >> 4, AK = (A_MN ? 2048 : 32) >> 4;
      constexpr u32 BL = (B_MN ? HG_K * 128 : S::B_BYTES) >> 4, BK = (B_MN ? 2048 : 32) >> 4;
      const u32 a0 = f16_desc_lo<A_MN>(base), b0 = f16_desc_lo<B_MN>(base + 2 * S::A_BYTES);
      u32 j = 0, s = 0, phase = 0, da = a0, db = b0;   // j counts chunks
      while (ok && work.next()) {
        for (u32 c = work.c0; ok && c < work.c1; ++c, ++j) {
          const u32 k1 = (c + 1) * CK < kbs ? CK : kbs - c * CK, buf = j & 1;
          if (j >= 2 && !wait(acce(buf), ((j >> 1) - 1) & 1, 5)) { ok = false; break; }
          tc_fence_after();
          const u32 acc = tmem + buf * S::ACCS * BN;
          for (u32 kb = 0; kb < k1; ++kb) {
            if (!wait(full(s), phase, 3)) { ok = false; break; }
            tc_fence_after();
            if (leader) {
#pragma unroll
              for (int k = 0; k < HG_K / 16; ++k) {
                const u32 ah = da + AK * k, al = ah + AL, bh = db + BK * k, bl = bh + BL;
                const bool on = k > 0 || kb != 0;
                if (S::ACCS == 1) {
                  mma_f16<CTAS, ID, AH, BH>(acc, al, bh, on);
                  mma_f16<CTAS, ID, AH, BH>(acc, ah, bl, true);
                  mma_f16<CTAS, ID, AH, BH>(acc, ah, bh, true);
                } else {
                  mma_f16<CTAS, ID, AH, BH>(acc + BN, al, bh, on);
                  mma_f16<CTAS, ID, AH, BH>(acc, ah, bh, on);
                  mma_f16<CTAS, ID, AH, BH>(acc + (S::ACCS - 1) * BN, ah, bl, S::ACCS == 2 || on);
                }
              }
              if constexpr (CTAS == 2) pair_commit(empty(s));
              else mma_commit(empty(s));
            }
            __syncwarp();
            da += S::STAGE >> 4;
            db += S::STAGE >> 4;
            if (++s == STAGES) { s = 0; phase ^= 1; da = a0; db = b0; }
          }
          if (ok && leader) {
            if constexpr (CTAS == 2) pair_commit(accf(buf));
            else mma_commit(accf(buf));
          }
          __syncwarp();
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 232;");
    constexpr int NB = BN / 64;   // 32-column blocks a warp
    F16Epi e;
    const int w = warp - 4;
    e.q = warp & 3;
    e.c0 = w / 4 * (BN / 2);
    e.lane = lane;
    e.M = M;
    e.N = N;
    e.stage = staging + (u32)w * 4096;
    e.gstage = gbase + (e.stage - base);
    e.vec = reinterpret_cast<float*>(gbase + (vectors - base)) + w * 32;
    epi.start(e.gstage - w * 4096);
    u32 j = 0;
    while (ok && work.next()) {
      e.T = f16_tile<BN, CTAS, SYM>(work.tile, tm, tn, per);
      e.T.m0 += (int)rank * HG_M;
      e.row = (u64)e.T.m0 + 32 * e.q + lane;
      epi.begin(e);   // its loads are on their way while the products run
      float v[NB][32];
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int i = 0; i < 32; ++i) v[b][i] = 0.0f;
      for (u32 c = work.c0; c < work.c1; ++c, ++j) {
        const u32 buf = j & 1;
        if (!mbar_wait(accf(buf), (j >> 1) & 1, err, 4)) { ok = false; break; }
        tc_fence_after();
        f16_collect<BN, 0>(v, tmem + buf * S::ACCS * BN + ((u32)(32 * e.q) << 16) + (u32)e.c0);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if constexpr (CTAS == 2)
            asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" :: "r"(in_leader(acce(buf))) : "memory");
          else
            asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" :: "r"(acce(buf)) : "memory");
        }
      }
      // this warp's part of the tile reaches into the output
      bool mine = ok && (u32)e.T.m0 + 32 * e.q < M && (u32)(e.T.n0 + e.c0) < N;
      if (mine && !work.whole()) {
        // CTA (or pair) c's slots: 2 c + 1 for the beginning of a tile, 2 c for a later part of one
        constexpr u64 SLOT = (u64)8 * NB * 1024 * CTAS;
        float* part = J.part + (u64)(8 * rank + w) * NB * 1024 + lane;
        f16_partial_store<0>(v, part + (2 * unit + (work.c0 == 0)) * SLOT);
        __threadfence();
        __syncwarp();
        const u64 first = (u64)(work.tile - work.full) * work.per;
        const u32 ca = work.owner(first), cb = work.owner(first + work.per - 1);
        u32* count = J.counters + ((work.tile - work.full) * CTAS + rank) * 8 + w;
        u32 old = 0;
        if (lane == 0) old = atomicAdd(count, 1u);
        old = __shfl_sync(0xffffffffu, old, 0);
        mine = old == cb - ca;
        if (mine) {
          __threadfence();
          f16_partial_load<false>(v, part + (2 * ca + 1) * SLOT);
#pragma unroll 1
          for (u32 c = ca + 1; c <= cb; ++c) f16_partial_load<true>(v, part + 2 * c * SLOT);
          if (lane == 0) *count = 0u;   // every part has arrived: zero for the next launch
        }
      }
      if (mine) {
        f16_blocks<0>(epi, e, v, N);
        epi.end(e);
      }
    }
    epi.done(e);
  }
  tc_fence_before();
  sync_settled(!ok);
  if constexpr (CTAS == 2) pair_sync();   // neither CTA ends, nor gives up its tensor memory, while the other works
  if (warp == 1) {
    tc_fence_after();
    if constexpr (CTAS == 2)
      asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" :: "r"(tmem), "r"(S::TMEM) : "memory");
    else
      asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" :: "r"(tmem), "r"(S::TMEM) : "memory");
  }
}

// a kernel's cluster by its CTAs a tile
#define TCB_F16_CLUSTER_1
#define TCB_F16_CLUSTER_2 __cluster_dims__(2, 1, 1)
// X(suffix of the names, BN, CTAS) for every tile
#define TCB_F16_TILES(X) X(256x2, 256, 2) X(128x2, 128, 2) X(128, 128, 1) X(64, 64, 1)

// ---- what the operators share ----

// Clears a launch's control block of n words (its first kernel does).
__device__ __forceinline__ void f16_clear(const Args& a, u32 n) {
  if (blockIdx.x == 0 && blockIdx.y == 0 && a.p[15])
    for (u32 i = threadIdx.x; i < n; i += blockDim.x) reinterpret_cast<u32*>(a.p[15])[i] = 0u;
}
constexpr u32 F16_CTRL = 4 + 8 * 2 * 148;   // words: the error word, 8 counters for each divided tile of two products

// 32 columns of hi / lo pairs through the warp's staging block to two planes of an fp16 array by TMA
// store (map: {cols, rows, planes}, boxes of 32 x 32 x 2, 64-byte swizzle).
__device__ __forceinline__ void stage_split32(const F16Epi& e, const float (&v)[32]) {
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
}
__device__ __forceinline__ void send_split32(const F16Epi& e, const TmaDesc* map, int col, int row, int matrix) {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  __syncwarp();
  if (e.lane == 0) {
    tma_store_3d(map, e.stage, col, row, 2 * matrix);
    bulk_commit();
  }
}

__device__ __forceinline__ void store_split32(const F16Epi& e, const TmaDesc* map, const float (&v)[32], int col, int row, int matrix) {
  stage_split32(e, v);
  send_split32(e, map, col, row, matrix);
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
      const float send = up ? v[j] : v[j + o];
      v[j] = up ? v[j + o] : v[j];
      v[j + o] = __shfl_xor_sync(0xffffffffu, send, o);
    }
#pragma unroll
    for (int j = 0; j + 1 < o; j += 2) add2(v[j], v[j + 1], v[j + o], v[j + o + 1]);
    if (o == 1) v[0] = __fadd_rn(v[0], v[1]);
  }
  return v[0];
}

}  // namespace tcb
