// Attention of a prompt chunk over the 8-bit cache on the fifth-generation tensor cores, causal, with an optional
// sliding window and sinks (the rule of al_q8_decode.cuh).
//
// The T x h query rows of a KV group are one list (row r = t * h + head), so all heads of a group share every key tile.
// A CTA takes 256 of them as two tiles of 128 rows (TMEM lanes; one tile where there are few) and walks the key tiles (128 tokens) that any of its
// rows can see, in steps of one block of the cache (64 tokens). Per step and query tile: S = Q K^T (tcgen05.mma, f16
// operands from shared memory, fp32 in TMEM), the softmax weights P go back into S's columns as f16, and O += P V (P
// from TMEM, V from shared memory). S has two buffers per query tile, so the next step's scores are there before this
// step's weights are done: the softmax warps do not wait for the tensor cores.
//   warps 0-3, 4-7  one thread per query row: scores -> running maximum, weights, denominator; O is rescaled only when
//                   a row's maximum grew by more than 2^8 (weights up to 2^14 fit f16)
//   warps 8-11      read the codes from global memory, convert them to f16 (exact) and store them in the 128-byte
//                   swizzled layout both contractions read; the next tile's codes are in registers meanwhile
//   warps 12, 13    issue the MMAs, one per query tile
// 16-bit queries are one f16 operand (scaled by a power of two per row, exact), and so are their weights: 11 bits, where the
// output is rounded to 8 (a second term would double the P V MMAs; against elementary fp32 operations rounded once, outputs
// move by 6.5e-4 in the norm, one ulp at most, and the error against 64 bits stays 1.6e-3). Denominators are summed from
// unrounded weights. 32-bit queries and their weights are split into two f16 terms (SPLIT): twice the MMAs, about 21 bits,
// one query tile a CTA (see kQpFlush). f16 ends either kind 2^-31 below a row's largest weight (see kQpBias).
//
// Bound: shared memory and the MUFU together. A step's MMAs read their operands for 1280 cycles of an SM's shared-
// memory bandwidth (Q again for every 64 keys), the converting warps store 32 KB (256 cycles), and its exponentials
// hold the MUFU pipe for 1024; measured are about 1800 a step. 8192 tokens of 32/8 heads: 520 us, 1.06 PFLOP/s of
// causal pairs, for the first 50 ms; then 565 under the power cap (SMs near 1800 MHz). 1024 tokens late in two 16K
// contexts with a window of 2048: 101 us (256 CTAs in two waves). Q K^T over 128 keys reads less but leaves one score
// buffer: 614 us.
//
// V codes that are NaN would reach rows that do not see them (0 * NaN in the MMA): they are replaced by zero on the way
// in, their tokens noted, and rows that do see one get their NaN in the epilogue.
#pragma once
#include "al_tcgen05.cuh"
#include "al_q8_decode.cuh"

namespace al {

constexpr int kQpRows = 128;                           // query rows per tile
constexpr int kQpKeys = 128;                           // tokens per key tile: two blocks of the cache
constexpr int kQpThreads = 512;
constexpr uint32_t kQpTile = kQpKeys * kHeadDim * 2;   // 32 KB: a tile of 128 x 128 f16, two 64-wide halves of 16 KB
constexpr uint32_t kQpHalf = kQpTile / 2;
constexpr int kQpPitch = 256 + 16;                     // output rows on their way out, 256 bytes at a time: no bank twice
constexpr uint32_t kQpStage = kQpRows * kQpPitch;      // 34 KB
static_assert(kQpStage % 1024 == 0, "tiles start on 1 KB");
constexpr size_t kQpSmem = 1024 + 4 * kQpTile + 2 * kQpStage;   // 2 Q + 2 K + 2 V tiles (a 32-bit tile's two terms are less)
constexpr int kQpNanList = 64;
// 32-bit queries: steps that O accumulates before it is added to the sum in TMEM's free half, in fp32 with rounding. The
// tensor cores cut each of their sums off towards zero: without this the output loses 2.3e-6 over 1024 tokens, 1.8e-5 over
// 16384 (elementary operations in fp32: 0.7e-6, 2.3e-6). 16-bit outputs are rounded to 2e-3 in any case (a sum cuts off
// about 1.3e-8: with one term 1.3e-5 over 16384 tokens of one CTA, 1e-4 over 131072).
constexpr int kQpFlush = 4;
// Weights run up to 2^(6 + 8), and f16's smallest step is 2^-24: a weight is good to 2^-31 of the row's largest at the worst.
// The largest is that of 2^(s + ev), so a block of V that is 2^31 quieter than a visible one leaves nothing in the output,
// also in dimensions where the loud block's codes are zero.
constexpr float kQpBias = 6.0f, kQpLazy = 8.0f;
// Registers a thread after the split: 2 x 128 softmax threads, 128 converting threads, the MMA warp's group.
// 184 + 184 + 104 + 40 = 512 = 4 x the 128 of the launch.
constexpr int kQpRegsSoftmax = 184, kQpRegsConvert = 104, kQpRegsMma = 40;

// Instruction descriptors (kind::f16): fp32 accumulator, f16 operands, M = 128; Q K^T has N = 64 (a block) and both
// operands K-major, P V has N = 128 (the head dimension) and V N-major.
constexpr uint32_t kQpIdescQK = (1u << 4) | ((uint32_t)(kQ8Block >> 3) << 17) | ((uint32_t)(kQpRows >> 4) << 24);
constexpr uint32_t kQpIdescPV = (1u << 4) | (1u << 16) | ((uint32_t)(kHeadDim >> 3) << 17) | ((uint32_t)(kQpRows >> 4) << 24);

// The MMA warp runs its loop with all lanes (waits, addresses and descriptors stay warp-uniform, so they live in uniform
// registers); `lead`, set in one lane, predicates the instructions one thread issues. With the loop inside a lane-0
// branch every MMA took two to four register moves and each wait about 300 cycles.
// Descriptors are passed as their low word (address and leading offset); the high word is the same for all tiles here.
constexpr uint32_t kQpDescHigh = (1024u >> 4) | (1u << 14) | (2u << 29);   // 8-row stride 1 KB, version 1, 128-byte swizzle
__device__ __forceinline__ void qp_mma_ss(uint32_t lead, uint32_t d, uint32_t a, uint32_t b, uint32_t accumulate) {
  asm volatile("{\n .reg .pred p, q;\n .reg .b64 da, db;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n"
               " mov.b64 da, {%1, %6};\n mov.b64 db, {%2, %6};\n"
               " @q tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n}\n"
               ::"r"(d), "r"(a), "r"(b), "r"(kQpIdescQK), "r"(accumulate), "r"(lead), "r"(kQpDescHigh) : "memory");
}
__device__ __forceinline__ void qp_mma_ts(uint32_t lead, uint32_t d, uint32_t a, uint32_t b, uint32_t accumulate) {
  asm volatile("{\n .reg .pred p, q;\n .reg .b64 db;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n"
               " mov.b64 db, {%2, %6};\n"
               " @q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n}\n"
               ::"r"(d), "r"(a), "r"(b), "r"(kQpIdescPV), "r"(accumulate), "r"(lead), "r"(kQpDescHigh) : "memory");
}
__device__ __forceinline__ void qp_commit(uint32_t lead, uint64_t* bar) {
  asm volatile("{\n .reg .pred q;\n setp.ne.b32 q, %1, 0;\n"
               " @q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}\n"
               ::"r"(smem_addr(bar)), "r"(lead) : "memory");
}
// Bounded wait for the phase with parity `parity`, small enough to be inlined everywhere (pf_wait's loop took 2 KB of
// code a place, and the warps of this kernel live off the instruction cache). Gives up like pf_wait.
__device__ __forceinline__ void qp_wait(uint64_t* bar, unsigned parity, volatile int* abort_flag, unsigned* err) {
  const uint32_t a = smem_addr(bar);
  uint32_t done;
  asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
               : "=r"(done) : "r"(a), "r"(parity) : "memory");
  if (done || *abort_flag) return;
  asm volatile("{\n .reg .pred p, q;\n .reg .u32 n;\n mov.u32 n, 0;\n"
               "WAIT:\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
               " add.u32 n, n, 1;\n setp.lt.and.u32 q, n, %3, !p;\n @q bra WAIT;\n"
               " selp.u32 %0, 1, 0, p;\n}\n"
               : "=r"(done) : "r"(a), "r"(parity), "r"((uint32_t)kWaitPolls) : "memory");
  if (!done) {
    *abort_flag = 1;
    atomicOr(err, kErrWaitLimit);
  }
}
__device__ __forceinline__ void qp_tmem_st32(uint32_t taddr, const uint32_t (&v)[32]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
               "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};\n"
               ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
                 "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]),
                 "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]),
                 "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
               : "memory");
}
// 64 consecutive TMEM columns of the thread's lane, defined on return.
__device__ __forceinline__ void qp_tmem_ld64(uint32_t taddr, uint32_t (&v)[64]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x64.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
               "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,"
               "%42,%43,%44,%45,%46,%47,%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63}, [%64];\n"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
                 "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]),
                 "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]),
                 "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31]),
                 "=r"(v[32]), "=r"(v[33]), "=r"(v[34]), "=r"(v[35]), "=r"(v[36]), "=r"(v[37]), "=r"(v[38]), "=r"(v[39]),
                 "=r"(v[40]), "=r"(v[41]), "=r"(v[42]), "=r"(v[43]), "=r"(v[44]), "=r"(v[45]), "=r"(v[46]), "=r"(v[47]),
                 "=r"(v[48]), "=r"(v[49]), "=r"(v[50]), "=r"(v[51]), "=r"(v[52]), "=r"(v[53]), "=r"(v[54]), "=r"(v[55]),
                 "=r"(v[56]), "=r"(v[57]), "=r"(v[58]), "=r"(v[59]), "=r"(v[60]), "=r"(v[61]), "=r"(v[62]), "=r"(v[63])
               : "r"(taddr) : "memory");
  tmem_wait_ld();
#pragma unroll
  for (int i = 0; i < 64; ++i) asm volatile("" : "+r"(v[i]));
}
// Asynchronous copy of `bytes` (a multiple of 16) from shared to global memory, both on 16-byte boundaries, and the wait
// until the sources of this thread's copies are read.
__device__ __forceinline__ void qp_bulk_store(const void* dst, uint32_t src, uint32_t bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;\n cp.async.bulk.commit_group;\n"
               ::"l"(__cvta_generic_to_global(dst)), "r"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void qp_bulk_read_wait() { asm volatile("cp.async.bulk.wait_group.read 0;\n" ::: "memory"); }
// Named barriers of a pair of warps: one waits, the other only arrives.
__device__ __forceinline__ void qp_bar_sync(int id) { asm volatile("bar.sync %0, 64;\n" ::"r"(id) : "memory"); }
__device__ __forceinline__ void qp_bar_arrive(int id) { asm volatile("bar.arrive %0, 64;\n" ::"r"(id) : "memory"); }
// The n lowest bits (n is clamped to [0, 64]).
__device__ __forceinline__ uint64_t qp_low_bits(int n) { return n >= 64 ? ~0ull : n <= 0 ? 0ull : (1ull << n) - 1ull; }
// Largest of three; a NaN gives way to a number.
__device__ __forceinline__ float qp_max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;\n" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ void qp_st_shared16(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};\n" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
__device__ __forceinline__ void qp_st_shared8(uint32_t a, uint32_t x, uint32_t y) {
  asm volatile("st.shared.v2.b32 [%0], {%1, %2};\n" ::"r"(a), "r"(x), "r"(y) : "memory");
}
__device__ __forceinline__ uint4 qp_ld_shared16(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ void qp_fence_async() { asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory"); }
// 16-byte chunk c (0..15, 8 f16 each) of row r in a 128-byte swizzled tile of two 64-wide halves.
__device__ __forceinline__ uint32_t qp_chunk(uint32_t tile, int r, int c) {
  return tile + (uint32_t)(c >> 3) * kQpHalf + (uint32_t)r * 128u + (uint32_t)(((c & 7) ^ (r & 7)) << 4);
}

template <bool B> struct QpFlag { static constexpr bool value = B; };
template <int I> struct QpInt { static constexpr int value = I; };

// TILES: query tiles of 128 rows a CTA takes, 2, or 1 where that spreads few rows over more CTAs.
template <typename T, int TILES>
__global__ void __launch_bounds__(kQpThreads, 1) q8_prompt_kernel(const Q8AttendParams p) {
  constexpr bool SPLIT = sizeof(T) == 4;
  static_assert(!SPLIT || TILES == 1, "the second tile's TMEM holds the sums of 32-bit queries");
  constexpr int NS = 2;                                // key tiles in flight
  constexpr int QP = SPLIT ? 2 : 1;                    // f16 terms per query row
  constexpr uint32_t QS = SPLIT ? 2 * kQpTile : kQpStage;   // bytes of a query tile, later of its output rows
  extern __shared__ __align__(1024) unsigned char qp_raw[];
  __shared__ uint64_t s_qfull[2], s_full[2][NS], s_empty[2][NS], s_sfull[2][2], s_pfull[2][2], s_pv[2][2];
  __shared__ uint32_t s_taddr;
  __shared__ float s_frow[2 * kQpRows];
  __shared__ int s_nan_count, s_nan[kQpNanList];
  __shared__ volatile int s_abort;

  // What steers the MMA warps is broadcast from lane 0, so that the compiler knows it to be the same in a warp and keeps
  // descriptors and branches in the uniform datapath (otherwise every MMA takes some 45 instructions).
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  const uint32_t base = (smem_addr(qp_raw) + 1023u) & ~1023u;
  const uint32_t s_q = base, s_k = base + TILES * QS, s_v = s_k + NS * kQpTile;

  // the longest row tiles first; all (batch, group) pairs of a row tile together
  const int BG = p.B * p.G, R = p.h * p.T;
  const int split = blockIdx.y;
  const int tile = p.row_tiles - 1 - (int)(blockIdx.x / (unsigned)BG), bg = (int)(blockIdx.x % (unsigned)BG);
  const int b = (int)((unsigned)bg / (unsigned)p.G), g = bg - b * p.G;
  const int length = q8_length(p.len, b);               // used after the set-up, which hides its latency
  const int r0 = tile * TILES * kQpRows;
  const int ntile = TILES == 2 && r0 + kQpRows < R ? 2 : 1;
  if (tid == 13 * 32) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_qfull[i], kQpRows);
      for (int k = 0; k < 2; ++k) {
        mbar_init(&s_sfull[i][k], 1);
        mbar_init(&s_pfull[i][k], kQpRows);
        mbar_init(&s_pv[i][k], 1);                       // P V of the even, the odd steps
      }
    }
    for (int i = 0; i < NS; ++i) {
      for (int kv = 0; kv < 2; ++kv) { mbar_init(&s_full[kv][i], 128); mbar_init(&s_empty[kv][i], ntile); }
    }
    mbar_init_fence();
    s_nan_count = 0;
    s_abort = 0;
  }
  if (warp == 12) { tmem_alloc(&s_taddr, 512); tmem_relinquish(); }

  // Query rows of warps 0-7, 16 pieces of 16 bytes a lane: LPR lanes a row, PER rows at a time. Asked for first, so
  // that they arrive while barriers and TMEM are set up.
  constexpr int LPR = kHeadDim * (int)sizeof(T) / 16, PER = 32 / LPR;
  const int qt = (warp >> 2) & 1, wrow0 = (warp & 3) * 32;   // warps 0-7: the query tile and the warp's first row in it
  uint4 raw[16];                                       // of these warps and of the converting ones
  auto load_rows = [&](int round) {
    const int rq = r0 + qt * kQpRows + wrow0 + 16 * PER * round + lane / LPR, left = R - rq;   // rows from this one on
    // rows PER apart: PER / h tokens and PER % h heads further, one token more where the head wraps
    const int t0 = q8_row_token(rq, p), dt = p.h == 1 ? PER : p.h == PER ? 1 : 0, dh = PER - dt * p.h;
    int head = rq - t0 * p.h;
    const T* src = static_cast<const T*>(p.q) + b * p.q_sb + g * p.q_sg + head * p.q_sh + t0 * p.q_st + V16<T>::n * (lane % LPR);
    const long long hop = dt * p.q_st + dh * p.q_sh, wrap = p.q_st - p.h * p.q_sh;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      raw[i] = make_uint4(0u, 0u, 0u, 0u);               // rows past the last are zeros and are not stored
      if (i * PER < left) raw[i] = __ldg(reinterpret_cast<const uint4*>(src));
      src += hop;
      head += dh;
      if (head >= p.h) { head -= p.h; src += wrap; }
    }
  };
  if (warp < 8 && qt < ntile) load_rows(0);
  tmem_fence_before_sync();
  __syncthreads();
  tmem_fence_after_sync();
  const uint32_t tm = __shfl_sync(0xffffffffu, s_taddr, 0);   // S0 | S1 | O0 | O1, 128 columns each

  int n = __shfl_sync(0xffffffffu, length, 0);
  if (n < 0 || n > p.C) {
    if (tid == 0) atomicOr(p.err, kErrQ8Range);
    n = max(0, min(n, p.C));
  }
  const int pbase = n - p.T;
  const int plo = pbase + q8_row_token(r0, p), phi = pbase + q8_row_token(min(r0 + TILES * kQpRows - 1, R - 1), p);
  const Q8Range rg = q8_range(plo, phi, p.window, p.sinks, kQpKeys);
  // (total < 2^24 and nsplit <= 148: the products fit 32 bits)
  const int it0 = (int)((unsigned)rg.total * (unsigned)split / (unsigned)p.nsplit);
  const int it1 = (int)((unsigned)rg.total * (unsigned)(split + 1) / (unsigned)p.nsplit);
  const int nt = it1 - it0;
  auto tile_token = [&](int it) { return (it < rg.ns ? it : rg.first + (it - rg.ns)) * kQpKeys; };

  // Converting warps: a tile is converted in two halves of 64 tokens, K's then V's; four halves are in flight in
  // registers (with two the loads' latency showed: 545 us for 8192 tokens of 32/8 heads against 526). A thread takes 8
  // codes of each 64-wide half of a row: 8 lanes read 64 contiguous bytes, and store the 8 chunks of one row of a swizzled
  // half, each in its own banks.
  const int rw = (warp & 3) * 4 + (lane >> 3), c8 = lane & 7;   // row within a group of 16, 8-code piece
  const long long off = (long long)bg * p.C * kHeadDim + 8 * c8;
  // half u of the walk: tile u / 4, K for u % 4 < 2, V after; into pieces 4 slot ...: rows rw + 16 i, dimensions 8 c8 ...
  // and 64 + 8 c8 ... . Rows past the length repeat the last one (their weights are zero; what matters is that they are
  // finite, see `store`).
  auto load = [&](int u, auto slot) {
    constexpr int at = 4 * decltype(slot)::value;
    if (u >= 4 * nt) return;
    const int t0 = tile_token(it0 + (u >> 2)) + kQ8Block * (u & 1), j0 = t0 + rw;
    const uint8_t* src = ((u & 2) ? p.vc : p.kc) + off;
    auto piece = [&](int i, const uint8_t* row) {
      const uint2 a = __ldg(reinterpret_cast<const uint2*>(row)), c = __ldg(reinterpret_cast<const uint2*>(row + 64));
      raw[at + i] = make_uint4(a.x, a.y, c.x, c.y);
    };
    if (t0 + kQ8Block <= n) {
      src += (long long)j0 * kHeadDim;
#pragma unroll
      for (int i = 0; i < 4; ++i) piece(i, src + 16 * i * kHeadDim);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) piece(i, src + (long long)min(j0 + 16 * i, n - 1) * kHeadDim);
    }
  };

  if (warp < 8) {
    // ---------------------------------------------------------------------------------------------- query rows
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(kQpRegsSoftmax));
    const int row = tid & 127;
    if (qt < ntile && nt > 0) {
      const int r = min(r0 + qt * kQpRows + row, R - 1);
      const int pos = pbase + q8_row_token(r, p);
      const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
      const uint32_t tS = tm + lanes + (uint32_t)qt * 128u, tO = tm + lanes + 256u + (uint32_t)qt * 128u;
      const uint32_t tA = tm + lanes + 384u;           // the sum of 32-bit queries
      const uint32_t qtile = s_q + (uint32_t)qt * QS;
      // Every row is scaled by a power of two into f16 (32-bit rows: two f16 terms) and goes to its places in the query
      // tile. Row maxima: each lane's over its pieces, then a transposing reduction that leaves piece i's row to lane i.
#pragma unroll 1
      for (int round = 0; round < 2 / PER; ++round) {
        if (round > 0) load_rows(round);
        uint32_t amax[16];                               // of the bits without the sign
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const uint4 x = raw[i];
          if constexpr (SPLIT) {
            amax[i] = max(max(x.x & 0x7fffffffu, x.y & 0x7fffffffu), max(x.z & 0x7fffffffu, x.w & 0x7fffffffu));
          } else {
            const uint32_t y = __vmaxu2(__vmaxu2(x.x & 0x7fff7fffu, x.y & 0x7fff7fffu),
                                        __vmaxu2(x.z & 0x7fff7fffu, x.w & 0x7fff7fffu));
            amax[i] = max(y << 16, y & 0xffff0000u);
          }
        }
#pragma unroll
        for (int o = 8; o > 0; o >>= 1)
#pragma unroll
          for (int i = 0; i < o; ++i) {
            const bool up = (lane & o) != 0;
            const uint32_t send = up ? amax[i] : amax[i + o], keep = up ? amax[i + o] : amax[i];
            amax[i] = max(keep, __shfl_xor_sync(0xffffffffu, send, o));
          }
        if constexpr (SPLIT) amax[0] = max(amax[0], __shfl_xor_sync(0xffffffffu, amax[0], 16));
        const int eq = q8_row_exponent(amax[0]);
        const float inv = q8_exp2i(-eq) * p.qsign;
        const int lr = wrow0 + 16 * PER * round + lane / LPR;   // row of piece 0
        s_frow[qt * kQpRows + lr + (lane & 15) * PER] = p.scale * q8_exp2i(eq);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float z = __shfl_sync(0xffffffffu, inv, i, 16);
          float y[V16<T>::n];
          unpack(raw[i], y, static_cast<const T*>(nullptr));
          if constexpr (SPLIT) {
            uint32_t hi[2], lo[2];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const float u = y[2 * k] * z, w = y[2 * k + 1] * z;
              hi[k] = q8_pack_half2(u, w);
              const float2 x = q8_half2_floats(hi[k]);
              lo[k] = q8_pack_half2(u - x.x, w - x.y);
            }
            const uint32_t at = qp_chunk(qtile, lr + i, lane >> 1) + 8u * (uint32_t)(lane & 1);
            qp_st_shared8(at, hi[0], hi[1]);
            qp_st_shared8(at + kQpTile, lo[0], lo[1]);
          } else {
            qp_st_shared16(qp_chunk(qtile, lr + 2 * i, lane & 15), q8_pack_half2(y[0] * z, y[1] * z),
                           q8_pack_half2(y[2] * z, y[3] * z), q8_pack_half2(y[4] * z, y[5] * z), q8_pack_half2(y[6] * z, y[7] * z));
          }
        }
      }
      qp_fence_async();
      pf_arrive(&s_qfull[qt]);
      __syncwarp();
      const float f_row = s_frow[qt * kQpRows + row];
      // positions of the warp's rows, for the test that a step needs no mask
      const int rw0 = r0 + qt * kQpRows + wrow0;
      const int wlo = pbase + q8_row_token(min(rw0, R - 1), p), whi = pbase + q8_row_token(min(rw0 + 31, R - 1), p);
      const signed char* keb = p.ke + (long long)bg * p.NB;
      const signed char* veb = p.ve + (long long)bg * p.NB;
      float m = -INFINITY, l = 0.0f;
      float m_sum = -INFINITY;                         // the maximum that the sum in TMEM is relative to
      int ev_top = -128;                               // largest V exponent met so far
      const int nsteps = 2 * nt;
      auto step_token = [&](int step) { return tile_token(it0 + (step >> 1)) + kQ8Block * (step & 1); };
      auto step_block = [&](int step) { return min(step_token(step) / kQ8Block, p.NB - 1); };

      // Scores of a step into registers, hidden ones -inf.
      auto fetch = [&](uint32_t (&s)[64], int step, int j0) {
        const int buf = step & 1;
        qp_wait(&s_sfull[qt][buf], (uint32_t)(step >> 1) & 1u, &s_abort, p.err);
        tmem_fence_after_sync();
        __syncwarp();
        qp_tmem_ld64(tS + 64u * (uint32_t)buf, s);
        const bool whole = j0 + kQ8Block - 1 <= wlo && (p.window == 0 || j0 > whi - p.window || j0 + kQ8Block <= p.sinks);
        if (!whole) {
          // the visible columns as bits: [0, last], less those at or below `left` that are no sinks
          const int last = pos - j0, left = p.window > 0 ? last - p.window : -1, sink = p.window > 0 ? p.sinks - j0 : 0;
          const uint64_t seen = qp_low_bits(last + 1) & (~qp_low_bits(left + 1) | qp_low_bits(sink));
          const uint32_t m0 = (uint32_t)seen, m1 = (uint32_t)(seen >> 32);
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            if (!(m0 & (1u << i))) s[i] = 0xff800000u;
            if (!(m1 & (1u << i))) s[32 + i] = 0xff800000u;
          }
        }
      };
      // The warps of the two query tiles that share a scheduler (w and w + 4) take turns with their exponentials: side
      // by side in the same phase both wait for the MUFU pipe and then leave it idle together (602 -> 587 us for 8192
      // tokens of 32/8 heads).
      const bool turns = ntile == 2;
      const int mine = 1 + (warp & 3) + 4 * qt, other = 1 + (warp & 3) + 4 * (1 - qt);
      if (turns && qt == 1) qp_bar_arrive(other);
      int ek = keb[step_block(0)], ev = veb[step_block(0)];
#pragma unroll 1
      for (int step = 0; step < nsteps; ++step) {
        const int buf = step & 1;
        uint32_t s[64];
        const float f = q8_factor(f_row, ek), fev = (float)ev;
        const int ev_now = ev;
        if (step + 1 < nsteps) {
          const int blk = step_block(step + 1);
          ek = keb[blk];
          ev = veb[blk];
        }
        const int j0 = step_token(step);
        fetch(s, step, j0);
        float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < 64; i += 4) {
          mx[0] = qp_max3(mx[0], __uint_as_float(s[i]), __uint_as_float(s[i + 1]));
          mx[1] = qp_max3(mx[1], __uint_as_float(s[i + 2]), __uint_as_float(s[i + 3]));
        }
        const float cand = fmaf(fmaxf(mx[0], mx[1]), f, fev);
        const bool grow = cand > m + kQpLazy;            // m = -inf: any visible score
        if (__any_sync(0xffffffffu, grow)) {
          const float alpha = grow ? q8_ex2(m - cand) : 1.0f;
          if (grow) {
            l = q8_rescale(l, m - cand);
            m = cand;
          }
          if (step > 0) {
            // O holds every earlier step. (This step's scores came after the P V two steps back, so the barrier's
            // phase is this one or the next.)
            qp_wait(&s_pv[qt][1 - buf], (uint32_t)((step - 1) >> 1) & 1u, &s_abort, p.err);
            tmem_fence_after_sync();
            __syncwarp();
#pragma unroll 1
            for (int c = 0; c < 8; ++c) {
              uint32_t o[16];
              tmem_ld16(tO + 16u * (uint32_t)c, o);
              tmem_wait_ld();
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                asm volatile("" : "+r"(o[i]));
                o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
              }
#pragma unroll
              for (int i = 0; i < 16; i += 2) tmem_st2(tO + 16u * (uint32_t)c + (uint32_t)i, o[i], o[i + 1]);
            }
          }
        }
        if (SPLIT && step > 0 && step % kQpFlush == 0) {
          // O's share so far joins the sum; this step's P V starts O anew (the wait is the one above)
          qp_wait(&s_pv[qt][1 - buf], (uint32_t)((step - 1) >> 1) & 1u, &s_abort, p.err);
          tmem_fence_after_sync();
          __syncwarp();
          tmem_wait_st();
          const float fa = m_sum == m ? 1.0f : q8_ex2(m_sum - m);
#pragma unroll 1
          for (int c = 0; c < 8; ++c) {
            uint32_t o[16], a[16];
            tmem_ld16(tO + 16u * (uint32_t)c, o);
            tmem_ld16(tA + 16u * (uint32_t)c, a);        // (what it holds before the first time is not used)
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              asm volatile("" : "+r"(o[i]), "+r"(a[i]));
              if (step > kQpFlush) o[i] = __float_as_uint(fmaf(__uint_as_float(a[i]), fa, __uint_as_float(o[i])));
            }
#pragma unroll
            for (int i = 0; i < 16; i += 2) tmem_st2(tA + 16u * (uint32_t)c + (uint32_t)i, o[i], o[i + 1]);
          }
          m_sum = m;
        }
        const float mref = (m == -INFINITY ? 0.0f : m) - kQpBias, add = fev - mref;
        ev_top = max(ev_top, ev_now);
        float far = 0.0f;
        const bool is_far = ev_top - ev_now > kQ8FarExp;
        if (is_far) {
          // the denominator's terms on their own (see kQ8FarExp), from the scores still in TMEM: a rare path, kept small
#pragma unroll 1
          for (int c = 0; c < 64; c += 8) {
            uint32_t x[8];
            tmem_ld8(tS + 64u * (uint32_t)buf + (uint32_t)c, x);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              asm volatile("" : "+r"(x[i]));
              if (q8_sees(pos, j0 + c + i, p.window, p.sinks)) far += q8_ex2(fmaf(__uint_as_float(x[i]), f, -mref));
            }
          }
        }
        if (turns) qp_bar_sync(mine);
        const float2 f2 = make_float2(f, f), add2 = make_float2(add, add);
        float2 sum = make_float2(0.0f, 0.0f);
        uint32_t w[32], lo[SPLIT ? 32 : 1];
#pragma unroll
        for (int i = 0; i < 64; i += 2) {
          const float2 x = __ffma2_rn(make_float2(__uint_as_float(s[i]), __uint_as_float(s[i + 1])), f2, add2);
          const float2 y = make_float2(q8_ex2(x.x), q8_ex2(x.y));
          sum = __fadd2_rn(sum, y);
          const uint32_t hw = q8_pack_half2(y.x, y.y);
          w[i / 2] = hw;
          if (SPLIT) {
            const float2 z = q8_half2_floats(hw);
            lo[SPLIT ? i / 2 : 0] = q8_pack_half2(y.x - z.x, y.y - z.y);
          }
        }
        if (turns && (qt == 0 || step + 1 < nsteps)) qp_bar_arrive(other);
        qp_tmem_st32(tS + 64u * (uint32_t)buf, w);
        if constexpr (SPLIT) qp_tmem_st32(tS + 64u * (uint32_t)buf + 32u, lo);
        // (the unit after the choice: inside it, the loop compiles to 3 % more time)
        l += (is_far ? far : (sum.x + sum.y) * q8_exp2i(-ev_now)) * kQ8Unit;
        tmem_wait_st();
        tmem_fence_before_sync();
        pf_arrive(&s_pfull[qt][buf]);
      }
      qp_wait(&s_pv[qt][1], (uint32_t)(nt - 1) & 1u, &s_abort, p.err);
      tmem_fence_after_sync();
      __syncwarp();
      // O through shared memory (the query tile's, now free): every thread puts its row there and hands it to the copy
      // engine, 256 bytes at a time (a CTA's epilogue takes 3900 cycles; with 16 lanes storing a row 4400)
      const int bad = s_nan_count;
      const uint8_t* vbase = p.vc + (long long)bg * p.C * kHeadDim;
      const bool part = p.part != nullptr;
      const bool wide = part || SPLIT;                   // 32-bit rows: 64 dimensions at a time
      const int rr = r0 + qt * kQpRows + row;
      const float unit = part ? 1.0f : kQ8Unit, z = part ? 1.0f : l == 0.0f ? 0.0f : 1.0f / l;
      const float fa = m_sum == m ? 1.0f : q8_ex2(m_sum - m);
      const uint32_t stage = qtile + (uint32_t)(row * kQpPitch);
      const int head = r - (pos - pbase) * p.h;          // row r of a group is token r / h, head r % h; partial results keep r
      char* dst = part ? reinterpret_cast<char*>(p.part + (((long long)split * BG + bg) * R + r) * kHeadDim)
                       : reinterpret_cast<char*>(static_cast<T*>(p.out) + (((long long)bg * p.h + head) * p.T + (pos - pbase)) * kHeadDim);
#pragma unroll 1
      for (int c = 0; c < 4; ++c) {
        uint32_t o[32];
        pf_tmem_ld32(tO + 32u * (uint32_t)c, o);
        pf_tmem_wait(o);
        if (SPLIT && nsteps > kQpFlush) {
          uint32_t a[32];
          pf_tmem_ld32(tA + 32u * (uint32_t)c, a);
          pf_tmem_wait(a);
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(fmaf(__uint_as_float(a[i]), fa, __uint_as_float(o[i])));
        }
        if (bad > 0) {
          // tokens with a NaN code in V: the listed ones, or all of this CTA's when the list ran over
          const int cnt = bad <= kQpNanList ? bad : nt * kQpKeys;
          for (int i = 0; i < cnt; ++i) {
            const int j = bad <= kQpNanList ? s_nan[i] : tile_token(it0 + i / kQpKeys) + i % kQpKeys;
            if (j >= n || !q8_sees(pos, j, p.window, p.sinks)) continue;
            const uint32_t* v = reinterpret_cast<const uint32_t*>(vbase + (long long)j * kHeadDim + 32 * c);
#pragma unroll
            for (int d = 0; d < 8; ++d) {
              const uint32_t bits = q8_nan_mask(v[d]);
#pragma unroll
              for (int k = 0; k < 4; ++k)
                if (bits & (0x80u << (8 * k))) o[4 * d + k] = 0x7fffffffu;
            }
          }
          __syncwarp();
        }
#pragma unroll
        for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * unit * z);
        if (wide) {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            qp_st_shared16(stage + 128u * (uint32_t)(c & 1) + 16u * (uint32_t)i, o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t h4[4];
#pragma unroll
            for (int k = 0; k < 4; ++k)
              h4[k] = pack_bf16x2(__uint_as_float(o[8 * i + 2 * k]), __uint_as_float(o[8 * i + 2 * k + 1]));
            qp_st_shared16(stage + 64u * (uint32_t)c + 16u * (uint32_t)i, h4[0], h4[1], h4[2], h4[3]);
          }
        }
        if (c == 3 || (wide && (c & 1))) {
          qp_fence_async();
          if (rr < R) qp_bulk_store(dst + (wide ? 128 * (c - 1) : 0), stage, 256u);
          qp_bulk_read_wait();                           // the place is used again, or the CTA ends
        }
      }
      if (part && rr < R) {
        float* ml = p.part_ml + (((long long)split * BG + bg) * R + rr) * 2;
        ml[0] = m;
        ml[1] = l;
      }
    } else if (qt < ntile && nt == 0) {
      // nothing to see for any row of this CTA: zeros, or an empty partial
      const int rr = r0 + qt * kQpRows + row;
      if (rr < R) {
        if (p.part) {
          float* ml = p.part_ml + (((long long)split * BG + bg) * R + rr) * 2;
          ml[0] = -INFINITY;
          ml[1] = 0.0f;
        } else {
          const int t = q8_row_token(rr, p), head = rr - t * p.h;
          T* dst = static_cast<T*>(p.out) + (((long long)bg * p.h + head) * p.T + t) * kHeadDim;
          const float z[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
          for (int c = 0; c < 16; ++c) q8_store8(dst + 8 * c, z);
        }
      }
    }
  } else if (warp < 12) {
    // ---------------------------------------------------------------------------------------------- codes -> f16 tiles
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(kQpRegsConvert));
    // Stores a half. For V, `nan` collects 0 * value (screening the codes took half again as many instructions): NaN
    // when there is a NaN code, and then the half is read again, the codes replaced by zeros and their tokens listed.
    load(0, QpInt<0>());
    load(1, QpInt<1>());
    load(2, QpInt<2>());
    load(3, QpInt<3>());
    const uint32_t at = qp_chunk(0, rw, c8);
    auto store = [&](uint32_t dst, auto slot, int u, auto is_v) {
      __half2 nan = __floats2half2_rn(0.0f, 0.0f);
      const __half2 zero = nan;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const uint4 x = raw[4 * decltype(slot)::value + i];
          const uint2 w = k ? make_uint2(x.z, x.w) : make_uint2(x.x, x.y);
          const uint32_t h[4] = {q8_decode_lo(w.x), q8_decode_hi(w.x), q8_decode_lo(w.y), q8_decode_hi(w.y)};
          qp_st_shared16(dst + at + (uint32_t)k * kQpHalf + (uint32_t)i * 2048u, h[0], h[1], h[2], h[3]);
          if (decltype(is_v)::value) {
#pragma unroll
            for (int d = 0; d < 4; ++d) nan = __hfma2(*reinterpret_cast<const __half2*>(&h[d]), zero, nan);
          }
        }
      const uint32_t bits = *reinterpret_cast<const uint32_t*>(&nan);
      if (!decltype(is_v)::value || (bits & 0x7fff7fffu) == 0u) return;
#pragma unroll 1
      for (int i = 0; i < 8; ++i) {
        const int j = tile_token(it0 + (u >> 2)) + kQ8Block * (u & 1) + rw + 16 * (i >> 1);
        uint2 w = *reinterpret_cast<const uint2*>(p.vc + off + (long long)min(j, n - 1) * kHeadDim + 64 * (i & 1));
        if ((q8_nan_mask(w.x) | q8_nan_mask(w.y)) == 0u) continue;
        if (j < n) {
          const int k = atomicAdd(&s_nan_count, 1);
          if (k < kQpNanList) s_nan[k] = j;
        }
        w = make_uint2(q8_drop_nan(w.x), q8_drop_nan(w.y));
        qp_st_shared16(dst + at + (uint32_t)(i & 1) * kQpHalf + (uint32_t)(i >> 1) * 2048u, q8_decode_lo(w.x),
                       q8_decode_hi(w.x), q8_decode_lo(w.y), q8_decode_hi(w.y));
      }
    };
    // two halves into one tile: wait for its place, convert, ask for what comes four halves later, hand over
    auto fill = [&](int u, auto is_v) {
      constexpr int kv = decltype(is_v)::value ? 1 : 0;
      const QpInt<2 * kv> first;
      const QpInt<2 * kv + 1> second;
      const int it = u >> 2, st = it % NS;
      const uint32_t tile = (kv ? s_v : s_k) + (uint32_t)st * kQpTile;
      qp_wait(&s_empty[kv][st], ((uint32_t)(it / NS) & 1u) ^ 1u, &s_abort, p.err);
      store(tile, first, u, is_v);
      load(u + 4, first);
      store(tile + kQ8Block * 128u, second, u + 1, is_v);
      load(u + 5, second);
      qp_fence_async();
      pf_arrive(&s_full[kv][st]);
    };
#pragma unroll 1
    for (int u = 0; u < 4 * nt; u += 4) {
      fill(u, QpFlag<false>());
      fill(u + 2, QpFlag<true>());
    }
  } else {
    // ---------------------------------------------------------------------------------------------- MMAs
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(kQpRegsMma));
    const int qt = warp - 12;
    if (qt < ntile && nt > 0) {
      uint32_t lead;
      asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(lead));
      // low descriptor words: address / 16, leading offset / 16 (1 where the K-major layout does not use it)
      const uint32_t dq = ((s_q + (uint32_t)qt * QS) >> 4) | (1u << 16), dk = (s_k >> 4) | (1u << 16),
                     dv = (s_v >> 4) | ((kQpHalf >> 4) << 16);
      const uint32_t tS = tm + (uint32_t)qt * 128u, tO = tm + 256u + (uint32_t)qt * 128u;
      // (The low terms go first, while the sums are small: that halves what is cut off, 0.95e-6 to 0.5e-6 of the output.)
      auto scores = [&](int step) {                     // S = Q K^T for one block of the key tile
        const uint32_t kb = (uint32_t)((step >> 1) % NS) * kQpTile + (uint32_t)(step & 1) * (kQ8Block * 128u);
#pragma unroll
        for (int term = 0; term < QP; ++term)
#pragma unroll
          for (int ks = 0; ks < 8; ++ks) {
            const uint32_t o = (uint32_t)(ks >> 2) * kQpHalf + (uint32_t)(ks & 3) * 32u;
            qp_mma_ss(lead, tS + (uint32_t)(step & 1) * 64u, dq + (((uint32_t)(QP - 1 - term) * kQpTile + o) >> 4),
                      dk + ((kb + o) >> 4), (term | ks) > 0 ? 1u : 0u);
          }
        qp_commit(lead, &s_sfull[qt][step & 1]);
      };
      auto values = [&](int step) {                     // O += P V over the same block
        const uint32_t vb = (uint32_t)((step >> 1) % NS) * kQpTile + (uint32_t)(step & 1) * (kQ8Block * 128u);
#pragma unroll
        for (int term = 0; term < QP; ++term)
#pragma unroll
          for (uint32_t ks = 0; ks < 4; ++ks)
            qp_mma_ts(lead, tO, tS + (uint32_t)(step & 1) * 64u + (uint32_t)(QP - 1 - term) * 32u + ks * 8u,
                      dv + ((vb + ks * 2048u) >> 4), ((SPLIT ? step % kQpFlush : step) | term | (int)ks) > 0 ? 1u : 0u);
        qp_commit(lead, &s_pv[qt][step & 1]);
      };
      qp_wait(&s_full[0][0], 0, &s_abort, p.err);
      qp_wait(&s_qfull[qt], 0, &s_abort, p.err);
      tmem_fence_after_sync();
      scores(0);
      scores(1);
      qp_commit(lead, &s_empty[0][0]);
#pragma unroll 1
      for (int it = 0; it < nt; ++it) {
        const bool more = it + 1 < nt;
        const uint32_t par = (uint32_t)it & 1u;
        qp_wait(&s_full[1][it % NS], (uint32_t)(it / NS) & 1u, &s_abort, p.err);
        qp_wait(&s_pfull[qt][0], par, &s_abort, p.err);
        tmem_fence_after_sync();
        values(2 * it);
        if (more) {
          // the scores of the next tile go where P was: MMAs of one thread run in order
          qp_wait(&s_full[0][(it + 1) % NS], (uint32_t)((it + 1) / NS) & 1u, &s_abort, p.err);
          tmem_fence_after_sync();
          scores(2 * it + 2);
        }
        qp_wait(&s_pfull[qt][1], par, &s_abort, p.err);
        tmem_fence_after_sync();
        values(2 * it + 1);
        qp_commit(lead, &s_empty[1][it % NS]);
        if (more) {
          scores(2 * it + 3);
          qp_commit(lead, &s_empty[0][(it + 1) % NS]);
        }
      }
    }
    __syncwarp();
  }
  tmem_fence_before_sync();
  __syncthreads();
  tmem_fence_after_sync();
  if (warp == 12) tmem_dealloc(tm, 512);
}

// Merge of the key splits: WPR warps per row share the splits, a lane per 4 dimensions, then meet in shared memory (8
// for many splits of few rows, a token's; 1 for few splits of many rows, a prompt's). Launched so that it may start while
// the splits still run; it waits for them first.
constexpr int kQmWarps = 8;
template <typename T, int WPR>
__global__ void __launch_bounds__(32 * kQmWarps) q8_merge_kernel(const Q8AttendParams p) {
  __shared__ float s_m[kQmWarps], s_l[kQmWarps];
  __shared__ __align__(16) float s_o[kQmWarps][kHeadDim];
  const int BG = p.B * p.G, R = p.h * p.T, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, d = 4 * lane;
  const int first = warp - warp % WPR, part = warp % WPR;  // the row's first warp; this warp takes splits part + WPR i
  const long long rows = (long long)BG * R, row = min((long long)blockIdx.x * (kQmWarps / WPR) + warp / WPR, rows - 1);
  asm volatile("griddepcontrol.wait;\n" ::: "memory");
  // the common maximum: a lane per split (nsplit <= 32 * WPR)
  const int mine = part + WPR * lane;
  // the first partial rows are asked for together with their maxima
  constexpr int kAhead = 8;
  float4 v[kAhead];
  auto fetch = [&](int i) {
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int s = part + WPR * (i + k);
      if (s < p.nsplit) v[k] = *reinterpret_cast<const float4*>(p.part + ((long long)s * rows + row) * kHeadDim + d);
    }
  };
  fetch(0);
  float2 ml = make_float2(-INFINITY, 0.0f);
  if (mine < p.nsplit) ml = *reinterpret_cast<const float2*>(p.part_ml + ((long long)mine * rows + row) * 2);
  float M = ml.x;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
  if (WPR > 1) {
    if (lane == 0) s_m[warp] = M;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WPR; ++w) M = fmaxf(M, s_m[first + w]);
  }
  const float wgt = q8_merge_weight(ml.y, ml.x, M);
  float L = q8_merge_l(ml.y, ml.x, M);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
  float4 a = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 1
  for (int i = 0; part + WPR * i < p.nsplit; i += kAhead) {
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const float e = __shfl_sync(0xffffffffu, wgt, (i + k) & 31);
      if (part + WPR * (i + k) < p.nsplit) q8_merge_add(a, e, v[k]);
    }
    fetch(i + kAhead);
  }
  if (WPR > 1) {
    *reinterpret_cast<float4*>(&s_o[warp][d]) = a;
    if (lane == 0) s_l[warp] = L;
    __syncthreads();
    if (part > 0) return;
#pragma unroll
    for (int w = 1; w < WPR; ++w) {
      const float4 x = *reinterpret_cast<const float4*>(&s_o[first + w][d]);
      a.x += x.x; a.y += x.y; a.z += x.z; a.w += x.w;
      L += s_l[first + w];
    }
  }
  const float inv = L == 0.0f ? 0.0f : 1.0f / L;
  // (B G R < 2^31)
  const int bg = (int)((unsigned)row / (unsigned)R), r = (int)row - bg * R, t = q8_row_token(r, p), head = r - t * p.h;
  T* dst = static_cast<T*>(p.out) + (((long long)bg * p.h + head) * p.T + t) * kHeadDim + d;
  q8_store4(dst, q8_divided(a, inv));
}

}  // namespace al
