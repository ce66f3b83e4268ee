// Attention of a few query columns (a decode step, or a short chunk: T * h columns per KV group) over the 8-bit cache, with
// an optional sliding window and first tokens (sinks) that stay visible.
//
// A query at position p sees the tokens j <= p with window = 0, or j > p - window, or j < sinks. A CTA holds 8 columns
// (query, head) of one (batch, group); its warps walk steps of 32 tokens and every warp keeps its own online softmax,
// so no warp waits for another until the end. A warp streams its steps' K and V rows (8 KB a step) through a ring of
// its own in shared memory with cp.async (16-byte chunks XOR-swizzled by row, rows past the end zero-filled) and reads
// them as 16 bytes a lane straight into the tensor-core fragments: both contractions may permute their summed index,
// their tokens and their dimensions freely, and the order is chosen so that no two lanes of a quarter warp share a
// bank. K and V codes become f16 exactly; q and the softmax weights are split into two f16 terms that occupy the two
// halves of the MMA's 16 rows (rows 0-7 high, 8-15 low), so 8 columns with about 21 bits each cost the same MMAs as 16
// columns with 11. (f16 ends the weights 2^-35 below a row's largest: what lies lower is lost to the output, not to the
// denominator, which is summed from the unrounded weights.) The block's exponents enter as 2^(ek) on the scores and as
// an addend ev inside the weights' exponent: weights are w = 2^(s + ev - m) with the running maximum m over s + ev, the
// output sums w * code, and the denominator sums w * 2^-ev.
//
// Bound: HBM reads of 256 bytes per visible token and group. The work of a segment is split over a cluster of CTAs
// whose partial (m, l, O) are merged through distributed shared memory, so one launch does the whole step; with so few
// segments that clusters of 16 leave SMs idle, or with requests of their own lengths, over runs of steps whose partials
// go through global memory to q8_merge_kernel. 32 requests of 16K to 32K tokens, 32/8 heads: 260 us, 6.2 TB/s, for the
// first 50 ms at 1965 MHz; then the power cap holds the SMs near 1750 MHz and it takes 285 to 304 (the conversions and
// MMAs are close behind the memory). 32 of 32K: 324 us, 6.6 TB/s, then 365 to 389; one of 128K: 50 us, 5.4 TB/s; one of
// 2048: 5.1 us, all latency (launch, length, rows, a step, merge). (bf16; graph replays of ten calls. The figures
// beside the other choices here and in q8_plan are such replays at the full clock.) Registers fed from global memory
// without the ring ran the first at 417 us: two CTAs of four warps an SM held too few bytes in flight.
#pragma once
#include <cuda_fp16.h>
#include "al_q8.cuh"

namespace al {

constexpr int kQ8TokenCols = 16;           // up to this many query rows per group always take this kernel
constexpr int kQ8FewCols = 128;            // up to this many do while (segments x groups of 8 rows x tokens) is at most
constexpr long long kQ8FewTokens = 1 << 18;   // this; the rest take the prompt kernel
constexpr int kQdWarps = 4;
constexpr int kQdThreads = 32 * kQdWarps;
constexpr int kQdCols = 8;                 // columns (query, head) per CTA
constexpr int kQdStep = 32;                // tokens per warp step (half a block: one exponent each for K and V)
constexpr int kQdChunk = 4096;             // tokens per CTA where requests have their own lengths
constexpr int kQdStages = 2;               // ring stages per warp
constexpr uint32_t kQdStageBytes = 2 * kQdStep * kHeadDim;           // 8 KB: K rows, then V rows
constexpr size_t kQdSmem = kQdWarps * kQdStages * kQdStageBytes;     // 64 KB
// 32-bit queries: steps of a warp that O accumulates before it is added to a sum in shared memory, in fp32 with rounding
// (its lanes' own places, 4 KB a warp). The tensor cores cut each of their sums off towards zero: over 131072 tokens that
// one CTA walks alone the output lost 2.7e-5 without this (which costs 2 %: 32 fp32 requests of 16K to 32K tokens 261 us to
// 267). 16-bit outputs are rounded to 2e-3 in any case.
constexpr int kQdFlush = 8;
template <typename T> constexpr size_t kQdSmemOf = kQdSmem + (sizeof(T) == 4 ? kQdWarps * kQdCols * kHeadDim * sizeof(float) : 0);
constexpr float kQdBias = 10.0f;           // weights run up to 2^10, so f16's normal range starts 2^-24 below the largest

struct Q8AttendParams {
  const void* q;                           // [B,G,h,T,128] (strides)
  long long q_sb, q_sg, q_sh, q_st;
  const uint8_t* kc;
  const uint8_t* vc;
  const signed char* ke;
  const signed char* ve;
  Q8Lengths len;
  int B, G, h, T, C, NB;
  int window, sinks;                       // window 0: every earlier token; sinks counts only with a window
  float scale;                             // |softmax scale| * log2 e; its sign is folded into q
  float qsign;
  void* out;                               // [B,G,h,T,128] contiguous
  // split of the key range over CTAs that write partial results (part null: none), and the prompt kernel's row tiles
  int nsplit, row_tiles;
  int chunk;                               // token kernel with nsplit > 1: steps per CTA
  uint32_t h_magic;                        // r / h = (r * h_magic) >> 32 for the row numbers used (h > 1)
  float* part;                             // [nsplit][B*G][R][128] unnormalised O, R = T * h
  float* part_ml;                          // [nsplit][B*G][R][2]
  unsigned* err;
};

// What rows with positions [plo, phi] can see, as steps of `unit` tokens: `ns` steps from token 0 (the sinks), then
// steps from `first` to the one that holds phi.
struct Q8Range {
  int ns, first, total;
};
__device__ __forceinline__ Q8Range q8_range(int plo, int phi, int window, int sinks, int unit) {
  Q8Range r = {0, 0, 0};
  if (phi < 0) return r;
  if (window > 0) {
    const int w0 = max(plo - window + 1, 0);
    r.ns = (min(sinks, w0) + unit - 1) / unit;
    r.first = max(w0 / unit, r.ns);
  }
  r.total = r.ns + max(phi / unit + 1 - r.first, 0);
  return r;
}
__device__ __forceinline__ bool q8_sees(int p, int j, int window, int sinks) {
  return j <= p && (window == 0 || j > p - window || j < sinks);
}

__device__ __forceinline__ float q8_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t q8_pack_half2(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
// D += A (16x16 f16, row) * B (16x8 f16, col) with fp32 accumulate.
__device__ __forceinline__ void mma_f16_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                              uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
               "{%0,%1,%2,%3};\n"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Any e4m3 NaN code (0x7f or 0xff) among the 4 bytes of w: non-zero.
__device__ __forceinline__ uint32_t q8_nan_mask(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }
// The codes of w with NaN replaced by zero.
__device__ __forceinline__ uint32_t q8_drop_nan(uint32_t w) { return w & ~((q8_nan_mask(w) >> 7) * 0xffu); }

// Power of two that brings a row's largest magnitude (its bits, finite) into [2^13, 2^14): the exponent eq with
// q = (q 2^-eq) 2^eq. A maximum that is zero,
// subnormal or non-finite gives 0 (a NaN or infinity then makes the row's output NaN).
__device__ __forceinline__ int q8_row_exponent(uint32_t amax_bits) {
  const int E = (int)(amax_bits >> 23);
  return E == 0 || E == 255 ? 0 : max(E - 127 - 13, -126);
}

// The weights of a block whose V exponent lies far below others can leave fp32's range although the block counts in the
// denominator (w = 2^(s + ev - m) with m set by a loud block): beyond this distance the denominator's terms 2^(s - m)
// are taken by their own exponentials. At 90 the terms that fast sums lose are below 2^-36 of the denominator.
constexpr int kQ8FarExp = 90;
// x * 2^d for d <= 0, in two steps: 2^d alone may underflow where the product does not. d = -inf gives 0 (x finite).
__device__ __forceinline__ float q8_rescale(float x, float d) {
  const float a = q8_ex2(0.5f * d);
  return x * a * a;
}

// Denominators are held in units of 2^11: a token counts its weight (2^6 to 2^14) times 2^-ev, with ev in [-100, 120], so
// 2^25 tokens stay below 2^128 (blocks of zeros have ev = -100, and a CTA may walk very many) and one above 2^-126. Outputs
// take the unit back before they are divided; both steps are exact.
constexpr float kQ8Unit = 1.0f / 2048.0f;

// Merging partials (m, l, O): the weight of one with maximum m under the common maximum M, and its share of the
// denominator. An empty partial has m = -inf and l = 0; one whose every score was NaN has m = -inf and l NaN. Only empty
// partials, whose O may not have been written, are left out (a negative weight): one whose weight underflows still brings
// the NaN of a V code that it saw, so that the result's NaN do not depend on how the tokens were split.
constexpr float kQ8Skip = -1.0f;
__device__ __forceinline__ float q8_merge_weight(float l, float m, float M) {
  return m == -INFINITY ? (l == 0.0f ? kQ8Skip : 1.0f) : q8_ex2(m - M);
}
__device__ __forceinline__ float4 q8_divided(float4 a, float inv) {
  return make_float4(a.x * kQ8Unit * inv, a.y * kQ8Unit * inv, a.z * kQ8Unit * inv, a.w * kQ8Unit * inv);
}
__device__ __forceinline__ void q8_merge_add(float4& a, float weight, const float4& v) {
  if (weight != kQ8Skip) { a.x += weight * v.x; a.y += weight * v.y; a.z += weight * v.z; a.w += weight * v.w; }
}
__device__ __forceinline__ float q8_merge_l(float l, float m, float M) { return m == -INFINITY ? l : q8_rescale(l, m - M); }

// Raw score -> log2 units for a block: a row's factor times 2^ek, kept positive and finite so that a hidden score
// (-inf) stays -inf.
__device__ __forceinline__ float q8_factor(float f_row, int ek) {
  return fminf(fmaxf(f_row * q8_exp2i(ek), 1.17549435e-38f), 3.0e38f);
}

__device__ __forceinline__ void q8_store4(float* p, float4 v) { *reinterpret_cast<float4*>(p) = v; }
__device__ __forceinline__ void q8_store4(__nv_bfloat16* p, float4 v) {
  *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16x2(v.x, v.y), pack_bf16x2(v.z, v.w));
}
// r / h for a query row.
__device__ __forceinline__ int q8_row_token(int r, const Q8AttendParams& p) {
  return p.h == 1 ? r : (int)__umulhi((uint32_t)r, p.h_magic);
}

// 16 bytes global -> shared, zeros when !in (nothing is read then).
__device__ __forceinline__ void qd_copy16(uint32_t dst, const void* src, bool in) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(in ? 16 : 0) : "memory");
}
__device__ __forceinline__ void qd_sts16(uint32_t a, float4 v) {
  asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};\n" ::"r"(a), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w) : "memory");
}
__device__ __forceinline__ uint4 qd_lds16(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
  return v;
}

// Two CTAs of four warps an SM (with clusters of two, 32 x 8 segments of 16K to 32K tokens: 296 us; three CTAs at 168
// registers, with spills, 366; one of eight warps 302).
template <typename T>
__global__ void __launch_bounds__(kQdThreads, 2) q8_decode_kernel(const Q8AttendParams p) {
  extern __shared__ __align__(1024) unsigned char qd_raw[];
  float4 (*s_o)[kQdCols][kHeadDim / 4] = reinterpret_cast<float4 (*)[kQdCols][kHeadDim / 4]>(qd_raw);   // after the loop
  __shared__ float s_m[kQdWarps][kQdCols], s_l[kQdWarps][kQdCols];
  __shared__ __align__(16) float4 s_in[kMaxCluster][kHeadDim / 4];   // partials that the cluster's CTAs send to this one
  __shared__ float2 s_in_ml[kMaxCluster];

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g8 = lane >> 2, t4 = lane & 3;
  const int bg = blockIdx.y, b = (int)((unsigned)bg / (unsigned)p.G), g = bg - b * p.G;
  const int cs = gridDim.x, rank = blockIdx.x;
  const bool clustered = !p.part && cs > 1;
  if (p.part) asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");   // the merge, which waits for the end of this grid
  if (clustered) asm volatile("barrier.cluster.arrive.relaxed.aligned;\n" ::: "memory");   // this CTA runs; waited for below
  const int R = p.h * p.T;
  int n = q8_length(p.len, b);
  // the query row, asked for before anything waits for the length
  const int col0 = blockIdx.z * kQdCols;
  const int col_last = min(col0 + kQdCols, R) - 1;
  const int mycol = min(col0 + g8, R - 1);               // columns past the end repeat the last one and are not stored
  const int mytok = q8_row_token(mycol, p);
  Raw8<T> raw[4];
  {
    const T* src = static_cast<const T*>(p.q) + b * p.q_sb + g * p.q_sg + (mycol - mytok * p.h) * p.q_sh + mytok * p.q_st;
#pragma unroll
    for (int i = 0; i < 4; ++i) raw[i].load(src + 64 * (i >> 1) + 16 * t4 + 8 * (i & 1));
  }
  if (n < 0 || n > p.C) {
    if (tid == 0) atomicOr(p.err, kErrQ8Range);
    n = max(0, min(n, p.C));
  }
  const int myp = n - p.T + mytok;                       // this thread's column: position
  const int plo = n - p.T + q8_row_token(col0, p), phi = n - p.T + q8_row_token(col_last, p);
  const Q8Range rg = q8_range(plo, phi, p.window, p.sinks, kQdStep);

  const uint8_t* kbase = p.kc + (long long)bg * p.C * kHeadDim;
  const uint8_t* vbase = p.vc + (long long)bg * p.C * kHeadDim;
  const signed char* keb = p.ke + (long long)bg * p.NB;
  const signed char* veb = p.ve + (long long)bg * p.NB;
  const uint32_t ring = smem_addr(qd_raw) + (uint32_t)warp * (kQdStages * kQdStageBytes);
  auto step_token = [&](int s) { return (s < rg.ns ? s : rg.first + (s - rg.ns)) * kQdStep; };
  // Copy a step: 8 lanes a row, 4 rows at a time; chunk c of row r goes to place c ^ (r & 7).
  const int crow = lane >> 3, cch = lane & 7;
  // steps of this warp: first, stride, end. A cluster's CTAs interleave; splits merged through global memory take a run of
  // steps each, of one length whatever the request's, so that short requests leave their CTAs to others at once.
  int step = p.part ? rank * p.chunk + warp : rank * kQdWarps + warp;
  const int W = p.part ? kQdWarps : cs * kQdWarps;
  // the last split takes whatever is left: the host's idea of the lengths sizes the runs, it does not bound them
  const int end = p.part && rank + 1 < cs ? min(rg.total, (rank + 1) * p.chunk) : rg.total;
  if (p.part && rank * p.chunk >= rg.total) {              // nothing for this split: an empty partial
    if (tid <= col_last - col0) {
      float* ml = p.part_ml + (((long long)rank * gridDim.y + bg) * R + col0 + tid) * 2;
      ml[0] = -INFINITY;
      ml[1] = 0.0f;
    }
    return;
  }
  auto copy = [&](int s, int stage) {
    if (s < end) {
      const int j0 = step_token(s) + crow;
      const uint32_t dst = ring + (uint32_t)stage * kQdStageBytes + (uint32_t)crow * kHeadDim;
      const long long at = (long long)j0 * kHeadDim + 16 * cch;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t d = dst + (uint32_t)i * 512u + (uint32_t)((cch ^ ((crow + 4 * i) & 7)) << 4);
        const bool in = j0 + 4 * i < n;
        qd_copy16(d, kbase + (in ? at + i * 512 : 0), in);
        qd_copy16(d + kQdStep * kHeadDim, vbase + (in ? at + i * 512 : 0), in);
      }
    }
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < kQdStages; ++i) copy(step + i * W, i);
  int ek = 0, ev = 0;
  if (step < end) {
    const int blk = step_token(step) / kQ8Block;
    ek = keb[blk];
    ev = veb[blk];
  }

  // q fragments: k-slots (2t, 2t+1 | 2t+8, 2t+9) of MMA ks hold dimensions 4 ks .. 4 ks + 3 of the thread's 16-byte
  // pieces [16 t, 16 t + 16) (ks < 4) and [64 + 16 t, ...) (ks >= 4)
  uint32_t qa[8][4];
  float f_row;                                           // 2^eq * scale: raw score -> log2 units (before 2^ek)
  {
    float x[32];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float y[8];
      raw[i].floats(y);
#pragma unroll
      for (int j = 0; j < 8; ++j) x[8 * i + j] = y[j] * p.qsign;
    }
    uint32_t amax = 0;
#pragma unroll
    for (int i = 0; i < 32; ++i) amax = max(amax, __float_as_uint(x[i]) & 0x7fffffffu);
    amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    const int eq = q8_row_exponent(amax);
    const float inv = q8_exp2i(-eq);
    f_row = p.scale * q8_exp2i(eq);
#pragma unroll
    for (int ks = 0; ks < 8; ++ks) {
      float hi[4], lo[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float y = x[4 * ks + j] * inv;
        hi[j] = __half2float(__float2half_rn(y));
        lo[j] = y - hi[j];
      }
      qa[ks][0] = q8_pack_half2(hi[0], hi[1]); qa[ks][2] = q8_pack_half2(hi[2], hi[3]);
      qa[ks][1] = q8_pack_half2(lo[0], lo[1]); qa[ks][3] = q8_pack_half2(lo[2], lo[3]);
    }
  }

  float o[16][4];                                        // O: rows g8 (high weights) and g8 + 8 (low), n-tile j
#pragma unroll
  for (int j = 0; j < 16; ++j) { o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.0f; }
  float m = -INFINITY, l = 0.0f;
  int ev_top = -128;                                     // largest V exponent met so far
  // 32-bit queries: the sum O joins every kQdFlush steps, relative to m_sum; piece i of the lane is O's columns 4 (i & 3) ...
  // of the row halves (i < 4: [0] and [2], else [1] and [3])
  constexpr bool WIDE = sizeof(T) == 4;
  const uint32_t sums = smem_addr(qd_raw) + (uint32_t)kQdSmem + (uint32_t)(warp * kQdCols * kHeadDim * 4 + lane * 16);
  float m_sum = -INFINITY;
  int since = 0;
  bool summed = false;
  auto piece = [&](int i) {
    const int j = 4 * (i & 3), r = i >> 2;
    return make_float4(o[j][r] + o[j][r + 2], o[j + 1][r] + o[j + 1][r + 2], o[j + 2][r] + o[j + 2][r + 2], o[j + 3][r] + o[j + 3][r + 2]);
  };
  auto plus_sum = [&](int i, float fa) {                 // piece i and what the sum holds of it
    float4 v = piece(i);
    if (summed) {
      const uint4 x = qd_lds16(sums + (uint32_t)i * 512u);
      v.x = fmaf(__uint_as_float(x.x), fa, v.x); v.y = fmaf(__uint_as_float(x.y), fa, v.y);
      v.z = fmaf(__uint_as_float(x.z), fa, v.z); v.w = fmaf(__uint_as_float(x.w), fa, v.w);
    }
    return v;
  };

  // Fragment addresses: K row of n index g8 is (g8 >> 1) + 4 (g8 & 1), its chunks t4 and t4 + 4; V row of k-slot 2t + u
  // is t4 + 4u, its chunk (the n index g8) (g8 >> 1) + 4 (g8 & 1).
  const int rho = (g8 >> 1) | ((g8 & 1) << 2);
  const uint32_t ka0 = (uint32_t)rho * 128u + (uint32_t)((t4 ^ rho) << 4), ka1 = ka0 ^ 64u;
  const uint32_t va0 = (uint32_t)t4 * 128u + (uint32_t)((rho ^ t4) << 4), va1 = (uint32_t)(t4 + 4) * 128u + (uint32_t)((rho ^ (t4 + 4)) << 4);
  int stage = 0;
#pragma unroll 1
  for (; step < end; step += W) {
    const int j0 = step_token(step);
    cp_async_wait<kQdStages - 1>();
    __syncwarp();
    const uint32_t kst = ring + (uint32_t)stage * kQdStageBytes, vst = kst + kQdStep * kHeadDim;
    // scores: 4 n-tiles of 8 tokens
    float s[8];
#pragma unroll
    for (int nt = 0; nt < 4; ++nt) {
      const uint4 k0 = qd_lds16(kst + ka0 + (uint32_t)nt * 1024u), k1 = qd_lds16(kst + ka1 + (uint32_t)nt * 1024u);
      float acc[2][4] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};   // two chains of four MMAs
      const uint32_t w[8] = {k0.x, k0.y, k0.z, k0.w, k1.x, k1.y, k1.z, k1.w};
#pragma unroll
      for (int ks = 0; ks < 8; ++ks)
        mma_f16_16816(acc[ks >> 2], qa[ks][0], qa[ks][1], qa[ks][2], qa[ks][3], q8_decode_lo(w[ks]), q8_decode_hi(w[ks]));
      s[2 * nt] = (acc[0][0] + acc[1][0]) + (acc[0][2] + acc[1][2]);
      s[2 * nt + 1] = (acc[0][1] + acc[1][1]) + (acc[0][3] + acc[1][3]);
    }
    const float f = q8_factor(f_row, ek), fev = (float)ev, inv_ev = q8_exp2i(-ev);
    const int ev_now = ev;
    if (step + W < end) {
      const int blk = step_token(step + W) / kQ8Block;
      ek = keb[blk];
      ev = veb[blk];
    }
    // a step is whole when every column sees all of it
    const bool whole = j0 + kQdStep - 1 <= plo && (p.window == 0 || j0 > phi - p.window || j0 + kQdStep <= p.sinks);
#pragma unroll
    for (int i = 0; i < 8; ++i) s[i] *= f;
    if (!whole) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int j = j0 + 8 * (i >> 1) + 4 * (i & 1) + t4;
        if (!q8_sees(myp, j, p.window, p.sinks)) s[i] = -INFINITY;
      }
    }
    float mx = s[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) mx = fmaxf(mx, s[i]);
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
    const float mn = fmaxf(m, mx + fev);
    if (__any_sync(0xffffffffu, mn > m)) {
      const float alpha = mn > m ? q8_ex2(m - mn) : 1.0f;   // m = -inf: 0
      l = mn > m ? q8_rescale(l, m - mn) : l;
#pragma unroll
      for (int j = 0; j < 16; ++j) { o[j][0] *= alpha; o[j][1] *= alpha; o[j][2] *= alpha; o[j][3] *= alpha; }
      m = mn;
    }
    const float ref = (m == -INFINITY ? 0.0f : m) - kQdBias - fev;
    float sum = 0.0f;
    uint32_t pa[2][4];
#pragma unroll
    for (int ks = 0; ks < 2; ++ks)
#pragma unroll
      for (int u = 0; u < 2; ++u) {                         // n-tile 2 ks + u: k-slots 2t, 2t+1 (u = 0) or 2t+8, 2t+9
        const float w0 = q8_ex2(s[4 * ks + 2 * u] - ref), w1 = q8_ex2(s[4 * ks + 2 * u + 1] - ref);
        sum += w0 + w1;
        const float h0 = __half2float(__float2half_rn(w0)), h1 = __half2float(__float2half_rn(w1));
        pa[ks][2 * u] = q8_pack_half2(h0, h1);
        pa[ks][2 * u + 1] = q8_pack_half2(w0 - h0, w1 - h1);
      }
    ev_top = max(ev_top, ev_now);
    if (ev_top - ev_now > kQ8FarExp) {
      sum = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) sum += q8_ex2(s[i] - (ref + fev));
      l += sum * kQ8Unit;
    } else {
      l += sum * kQ8Unit * inv_ev;
    }
    uint4 vr[8];                                            // row 16 (i >> 2) + 8 (i >> 1 & 1) + 4 (i & 1) + t4
#pragma unroll
    for (int i = 0; i < 8; ++i) vr[i] = qd_lds16(vst + ((i & 1) ? va1 : va0) + (uint32_t)(i >> 1) * 1024u);
    __syncwarp();
    copy(step + kQdStages * W, stage);
    if (++stage == kQdStages) stage = 0;
    // O += P V. Rows that no column sees become zero codes. A NaN code in a row that only some columns see must not
    // reach the others (0 * NaN): such codes become zero too, and the columns that see them get their NaN here.
    if (!whole) {
      uint32_t bad = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int j = j0 + 8 * (i >> 1) + 4 * (i & 1) + t4;
        const bool none = j > phi || (p.window > 0 && j <= plo - p.window && j >= p.sinks);
        if (none) vr[i] = make_uint4(0, 0, 0, 0);
        bad |= q8_nan_mask(vr[i].x) | q8_nan_mask(vr[i].y) | q8_nan_mask(vr[i].z) | q8_nan_mask(vr[i].w);
      }
      if (plo != phi && __any_sync(0xffffffffu, bad != 0)) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          vr[i].x = q8_drop_nan(vr[i].x); vr[i].y = q8_drop_nan(vr[i].y);
          vr[i].z = q8_drop_nan(vr[i].z); vr[i].w = q8_drop_nan(vr[i].w);
        }
#pragma unroll 1
        for (int j = j0; j < min(j0 + kQdStep, n); ++j) {
          if (!q8_sees(myp, j, p.window, p.sinks)) continue;
          const uint8_t* v = vbase + (long long)j * kHeadDim + 16 * t4;
#pragma unroll
          for (int d = 0; d < 16; ++d) {
            if ((v[d] & 0x7f) == 0x7f) o[d][0] = __uint_as_float(0x7fffffffu);
            if ((v[64 + d] & 0x7f) == 0x7f) o[d][1] = __uint_as_float(0x7fffffffu);
          }
        }
        __syncwarp();
      }
    }
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      const uint4 a0 = vr[4 * ks], a1 = vr[4 * ks + 1], b0 = vr[4 * ks + 2], b1 = vr[4 * ks + 3];
      const uint32_t x0[4] = {a0.x, a0.y, a0.z, a0.w}, x1[4] = {a1.x, a1.y, a1.z, a1.w};
      const uint32_t y0[4] = {b0.x, b0.y, b0.z, b0.w}, y1[4] = {b1.x, b1.y, b1.z, b1.w};
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const uint32_t xl = __byte_perm(x0[w], x1[w], 0x5140), xh = __byte_perm(x0[w], x1[w], 0x7362);
        const uint32_t yl = __byte_perm(y0[w], y1[w], 0x5140), yh = __byte_perm(y0[w], y1[w], 0x7362);
        mma_f16_16816(o[4 * w], pa[ks][0], pa[ks][1], pa[ks][2], pa[ks][3], q8_decode_lo(xl), q8_decode_lo(yl));
        mma_f16_16816(o[4 * w + 1], pa[ks][0], pa[ks][1], pa[ks][2], pa[ks][3], q8_decode_hi(xl), q8_decode_hi(yl));
        mma_f16_16816(o[4 * w + 2], pa[ks][0], pa[ks][1], pa[ks][2], pa[ks][3], q8_decode_lo(xh), q8_decode_lo(yh));
        mma_f16_16816(o[4 * w + 3], pa[ks][0], pa[ks][1], pa[ks][2], pa[ks][3], q8_decode_hi(xh), q8_decode_hi(yh));
      }
    }
    if (WIDE && ++since == kQdFlush) {
      const float fa = m_sum == m ? 1.0f : q8_ex2(m_sum - m);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float4 v = plus_sum(i, fa);
        qd_sts16(sums + (uint32_t)i * 512u, v);
      }
#pragma unroll
      for (int j = 0; j < 16; ++j) { o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.0f; }
      m_sum = m;
      since = 0;
      summed = true;
    }
  }
  cp_async_wait<0>();
  __syncthreads();                                          // the rings give way to the partial results

  // The warps' partials in shared memory: thread holds column g8, dimensions 16 t + j (o[j][0] + o[j][2]: pieces 0-3) and
  // 64 + 16 t + j (pieces 4-7). Piece x (4 dimensions) of column c lies at x ^ (x >> 3 & 1) ^ 2 (c & 1): no bank twice.
  auto place = [](int c, int x) { return x ^ ((x >> 3) & 1) ^ ((c & 1) << 1); };
  l += __shfl_xor_sync(0xffffffffu, l, 1);
  l += __shfl_xor_sync(0xffffffffu, l, 2);
  const float fa = m_sum == m ? 1.0f : q8_ex2(m_sum - m);
#pragma unroll
  for (int i = 0; i < 8; ++i) s_o[warp][g8][place(g8, 16 * (i >> 2) + 4 * t4 + (i & 3))] = WIDE ? plus_sum(i, fa) : piece(i);
  if (t4 == 0) { s_m[warp][g8] = m; s_l[warp][g8] = l; }
  __syncwarp();
  if (clustered) asm volatile("barrier.cluster.wait.aligned;\n" ::: "memory");   // every CTA of the cluster runs
  __syncthreads();
  auto emit = [&](int c, float4 a, float L) {              // 4 dimensions of a finished column
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
    if (L == 0.0f) a = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    const int t = q8_row_token(col0 + c, p), hd = col0 + c - t * p.h;
    T* dst = static_cast<T*>(p.out) + (((long long)bg * p.h + hd) * p.T + t) * kHeadDim + 4 * lane;
    q8_store4(dst, q8_divided(a, inv));
  };
  // Merge. Every warp has all 32 (warp, column) weights, one a lane, and takes columns warp, warp + kQdWarps: a lane 4
  // dimensions. (With the weights worked out by every thread for itself, in 32 copies of the code, this took 4600 cycles.)
  const int ncol = col_last - col0 + 1;
  float M, L, e;
  {
    static_assert(kQdWarps * kQdCols == 32, "a lane per (warp, column)");
    const float mw = s_m[lane >> 3][lane & 7], lw = s_l[lane >> 3][lane & 7];
    M = fmaxf(mw, __shfl_xor_sync(0xffffffffu, mw, 8));
    M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, 16));
    e = q8_merge_weight(lw, mw, M);
    L = q8_merge_l(lw, mw, M);
    L += __shfl_xor_sync(0xffffffffu, L, 8);
    L += __shfl_xor_sync(0xffffffffu, L, 16);
  }
#pragma unroll 1
  for (int c = warp; c < ncol; c += kQdWarps) {
    float4 a = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int w = 0; w < kQdWarps; ++w) {
      const float ew = __shfl_sync(0xffffffffu, e, 8 * w + c);
      q8_merge_add(a, ew, s_o[w][c][place(c, lane)]);
    }
    const float Mc = __shfl_sync(0xffffffffu, M, c), Lc = __shfl_sync(0xffffffffu, L, c);
    if (p.part) {
      const long long row = ((long long)rank * gridDim.y + bg) * R + col0 + c;
      *reinterpret_cast<float4*>(p.part + row * kHeadDim + 4 * lane) = a;
      if (lane == 0) *reinterpret_cast<float2*>(p.part_ml + row * 2) = make_float2(Mc, Lc);
    } else if (cs == 1) {
      emit(c, a, Lc);
    } else {
      // to the CTA that finishes the column: rank c mod cs (cs is a power of two)
      const int owner = c & (cs - 1), slot = (c - owner) + rank;
      cg::cluster_group cluster = cg::this_cluster();
      *cluster.map_shared_rank(&s_in[slot][lane], owner) = a;
      if (lane == 0) *cluster.map_shared_rank(&s_in_ml[slot], owner) = make_float2(Mc, Lc);
    }
  }
  __syncwarp();
  if (!clustered) return;
  // One barrier, and every CTA finishes its columns from its own shared memory. (Reading the others' partials instead takes
  // a remote round trip and a second barrier.)
  asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;\n" ::: "memory");
#pragma unroll 1
  for (int c = rank + cs * warp; c < ncol; c += cs * kQdWarps) {
    const float2 ml = lane < cs ? s_in_ml[c - rank + lane] : make_float2(-INFINITY, 0.0f);
    M = ml.x;
#pragma unroll
    for (int o2 = 8; o2 > 0; o2 >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o2));
    e = q8_merge_weight(ml.y, ml.x, M);
    L = q8_merge_l(ml.y, ml.x, M);
#pragma unroll
    for (int o2 = 8; o2 > 0; o2 >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o2);
    L = __shfl_sync(0xffffffffu, L, 0);
    float4 a = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
    for (int r = 0; r < cs; ++r) {
      const float er = __shfl_sync(0xffffffffu, e, r);
      q8_merge_add(a, er, s_in[c - rank + r][lane]);
    }
    emit(c, a, L);
  }
}

}  // namespace al
