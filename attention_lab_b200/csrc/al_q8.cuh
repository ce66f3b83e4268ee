// The 8-bit cache: its format, rotary positions, the quantising write and the read-back.
//
// Format. One layer's K (and V alike) is a table of e4m3 codes [B,G,C,128] and, for every block of 64 tokens of every
// (batch, group), one int8 exponent e [B,G,ceil(C/64)]: value = code * 2^e. e is the smallest exponent with
// amax <= 448 * 2^e over the block's finite values, clamped to [-100, 120]; a NaN or an infinity is stored as the NaN
// code and does not count. Why a power of two: multiplying by it is exact, so a value is rounded once, when it is
// written; when a later token of the block raises e, the codes already there are shifted exactly except where they
// enter e4m3's subnormals, and the attention kernels fold e into the softmax exponent instead of multiplying rows.
#pragma once
#include "al_common.cuh"

namespace al {

constexpr int kQ8Block = 64;               // tokens per exponent
constexpr int kQ8EMin = -100, kQ8EMax = 120;
constexpr unsigned kErrQ8Range = 4u;       // a length outside [0, C] was clamped, or a position past the rotary table

// Lengths of the requests after this step's tokens: per_batch[b], or `all` when per_batch is null.
struct Q8Lengths {
  const int* per_batch;
  int all;
};
__device__ __forceinline__ int q8_length(const Q8Lengths& l, int b) { return l.per_batch ? l.per_batch[b] : l.all; }

__device__ __forceinline__ float q8_exp2i(int e) {   // 2^e, e clamped to the normal range
  return __int_as_float((max(-126, min(127, e)) + 127) << 23);
}

// Smallest e with amax <= 448 * 2^e for a non-negative finite amax given by its bits (448 = 1.75 * 2^8): the binade of
// amax less 8, one more when its fraction is above 1.75.
__device__ __forceinline__ int q8_exponent(uint32_t amax_bits) {
  if (amax_bits == 0u) return kQ8EMin;
  const int e = (int)(amax_bits >> 23) - 135 + ((amax_bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return max(kQ8EMin, min(kQ8EMax, e));
}

__device__ __forceinline__ bool q8_finite(float x) { return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u; }

// Two values to two codes (lo in the low byte), round to nearest even, NaN to the NaN code.
__device__ __forceinline__ uint32_t q8_encode2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;\n" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
// The two codes in the low / high half of w as f16x2 (exact: e4m3 is a subset of f16).
__device__ __forceinline__ uint32_t q8_decode_lo(uint32_t w) {
  uint32_t r;
  asm("{\n .reg .b16 a, b;\n mov.b32 {a, b}, %1;\n cvt.rn.f16x2.e4m3x2 %0, a;\n}\n" : "=r"(r) : "r"(w));
  return r;
}
__device__ __forceinline__ uint32_t q8_decode_hi(uint32_t w) {
  uint32_t r;
  asm("{\n .reg .b16 a, b;\n mov.b32 {a, b}, %1;\n cvt.rn.f16x2.e4m3x2 %0, b;\n}\n" : "=r"(r) : "r"(w));
  return r;
}
__device__ __forceinline__ float2 q8_half2_floats(uint32_t h) {
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

// 8 values times `scale` to 8 codes, and back to floats.
__device__ __forceinline__ uint2 q8_encode8(const float (&x)[8], float scale) {
  float y[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) y[j] = __fmul_rn(x[j], scale);
  return make_uint2(q8_encode2(y[0], y[1]) | (q8_encode2(y[2], y[3]) << 16),
                    q8_encode2(y[4], y[5]) | (q8_encode2(y[6], y[7]) << 16));
}
__device__ __forceinline__ void q8_decode8(const uint2& w, float (&x)[8]) {
  const float2 a = q8_half2_floats(q8_decode_lo(w.x)), b = q8_half2_floats(q8_decode_hi(w.x));
  const float2 c = q8_half2_floats(q8_decode_lo(w.y)), d = q8_half2_floats(q8_decode_hi(w.y));
  x[0] = a.x; x[1] = a.y; x[2] = b.x; x[3] = b.y; x[4] = c.x; x[5] = c.y; x[6] = d.x; x[7] = d.y;
}

// 8 elements of T as floats.
__device__ __forceinline__ void q8_load8(const __nv_bfloat16* p, float (&f)[8]) {
  unpack(*reinterpret_cast<const uint4*>(p), f, p);
}
__device__ __forceinline__ void q8_load8(const float* p, float (&f)[8]) {
  unpack(reinterpret_cast<const uint4*>(p)[0], f, p);
  unpack(reinterpret_cast<const uint4*>(p)[1], f + 4, p);
}
// 8 elements as they lie in memory (what a load in flight occupies), and as floats.
template <typename T> struct Raw8 {
  uint4 v[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) v[i] = reinterpret_cast<const uint4*>(p)[i];
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) v[i] = make_uint4(0, 0, 0, 0);
  }
  __device__ __forceinline__ void floats(float (&f)[8]) const {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) unpack(v[i], f + i * V16<T>::n, static_cast<const T*>(nullptr));
  }
};
__device__ __forceinline__ void q8_store8(__nv_bfloat16* p, const float (&f)[8]) {
  *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]),
                                            pack_bf16x2(f[6], f[7]));
}
__device__ __forceinline__ void q8_store8(float* p, const float (&f)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
}

// ------------------------------------------------------------------------------------------------ rotary positions
// Pair (a, b) -> (a c - b s, b c + a s) with c, s from the table row of the position (cosines, then sines; any factor
// on them is part of the table). Pairs are dimensions (i, i + rot/2) (half) or (2i, 2i + 1) (interleaved); dimensions
// from rot on pass through. Each product and sum is rounded on its own, so a rotation fused into the quantising write
// gives the codes of rotating in 32 bits first, bit for bit.
constexpr int kRotHalf = 0, kRotInterleaved = 1;

struct RotTable {
  const float* table;   // [rows, rot]
  int rows, rot, layout;
};

__device__ __forceinline__ void rot_pair(float& a, float& b, float c, float s) {
  const float x = __fsub_rn(__fmul_rn(a, c), __fmul_rn(b, s));
  b = __fadd_rn(__fmul_rn(b, c), __fmul_rn(a, s));
  a = x;
}

// A thread's share of a row's rotation: one item of 8 dimensions (or a pair of items half the rotated width apart),
// with its cosines and sines in registers while it walks over heads, which all share them. How a row splits into items:
//   kRotPairs   half layout, rot a multiple of 16: items 0 .. rot/16 - 1 are the dimension pairs [8 i, 8 i + 8) and
//               [rot/2 + 8 i, ...), each read once; the others are 8 dimensions past rot, copied
//   kRotInner   interleaved: 8 dimensions hold their own 4 pairs
//   kRotOdd     half layout, other rot: 8 dimensions, partners read one by one from the row (it is in L1 by then)
constexpr int kRotPairs = 0, kRotInner = 1, kRotOdd = 2;
__host__ __device__ __forceinline__ int rot_mode(int rot, int layout) {
  return layout == kRotInterleaved ? kRotInner : (rot % 16 == 0 ? kRotPairs : kRotOdd);
}
__host__ __device__ __forceinline__ int rot_items(int d, int rot, int mode) {   // items of a row
  return mode == kRotPairs ? (d - rot) / 8 + rot / 16 : d / 8;
}

template <int MODE>
struct RotItem {
  float c[8], s[8];           // kRotInner: 4 of each
  int d0, d1;                 // first dimension; of the second chunk (kRotPairs), or -1
  int live;                   // dimensions from d0 on that are rotated (0: copied)

  __device__ __forceinline__ void init(const RotTable& rt, const float* tr, int item, float sgn) {
    const int half = rt.rot >> 1;
    d1 = -1;
    if (MODE == kRotPairs) {
      const int pairs = rt.rot >> 4;
      d0 = item < pairs ? 8 * item : rt.rot + 8 * (item - pairs);
      live = item < pairs ? 8 : 0;
      if (live) {
        d1 = d0 + half;
#pragma unroll
        for (int i = 0; i < 8; i += 4) {
          const float4 x = __ldg(reinterpret_cast<const float4*>(tr + d0 + i));
          const float4 y = __ldg(reinterpret_cast<const float4*>(tr + half + d0 + i));
          c[i] = x.x; c[i + 1] = x.y; c[i + 2] = x.z; c[i + 3] = x.w;
          s[i] = sgn * y.x; s[i + 1] = sgn * y.y; s[i + 2] = sgn * y.z; s[i + 3] = sgn * y.w;
        }
      }
      return;
    }
    d0 = 8 * item;
    live = max(0, min(8, rt.rot - d0));
#pragma unroll
    for (int i = 0; i < (MODE == kRotInner ? 4 : 8); ++i) {
      const int pi = MODE == kRotInner ? (d0 >> 1) + i : (d0 + i < half ? d0 + i : d0 + i - half);
      const bool on = (MODE == kRotInner ? 2 * i : i) < live;
      c[i] = on ? __ldg(tr + pi) : 1.0f;
      s[i] = on ? sgn * __ldg(tr + half + pi) : 0.0f;
    }
  }
  // x: the chunk at d0; y: the chunk at d1 (kRotPairs). row: the row in memory (kRotOdd's partners).
  template <typename T>
  __device__ __forceinline__ void turn(float (&x)[8], float (&y)[8], const T* row, const RotTable& rt) const {
    if (MODE == kRotPairs) {
      if (!live) return;
#pragma unroll
      for (int i = 0; i < 8; ++i) rot_pair(x[i], y[i], c[i], s[i]);
    } else if (MODE == kRotInner) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (2 * i < live) rot_pair(x[2 * i], x[2 * i + 1], c[i], s[i]);
    } else {
      const int half = rt.rot >> 1;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (i >= live) continue;
        const bool low = d0 + i < half;
        const float z = tof(row[low ? d0 + i + half : d0 + i - half]);
        x[i] = low ? __fsub_rn(__fmul_rn(x[i], c[i]), __fmul_rn(z, s[i])) : __fadd_rn(__fmul_rn(x[i], c[i]), __fmul_rn(z, s[i]));
      }
    }
  }
};

// Rows of one tensor [B, H, T, d] (element strides sb, sh, st; last dimension contiguous) to a contiguous output.
struct RotTensor {
  const void* x;
  long long sb, sh, st;
  int H;
  void* out;
};

struct RotaryParams {
  RotTensor q, k;             // k.H = 0 when there is no second tensor
  RotTable rt;
  const long long* pos;       // [B, T] (strides pos_sb, pos_st), or null: start + t
  long long pos_sb, pos_st;
  long long start;
  int B, T, d;
  int items;                  // items of a row (rot_items)
  int hpt;                    // heads per thread
  float sgn;                  // -1: the inverse rotation (the gradient)
  unsigned* err;
};

// Heads [h0, h1) of one tensor at (b, t): U rows in flight. `in`: the position is in the table (else zeros).
template <typename T, int MODE, int U>
__device__ __forceinline__ void rot_heads(const RotTensor& x, int h0, int h1, int b, int t, int Tn, int d,
                                          const RotItem<MODE>& it, const RotTable& rt, bool in) {
  const T* src = static_cast<const T*>(x.x) + b * x.sb + t * x.st;
  T* dst = static_cast<T*>(x.out) + ((long long)b * x.H * Tn + t) * d;
  for (int h = h0; h < h1; h += U) {
    Raw8<T> v[U], w[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      v[u].zero();
      w[u].zero();
      if (in && h + u < h1) {
        v[u].load(src + (h + u) * x.sh + it.d0);
        if (MODE == kRotPairs && it.d1 >= 0) w[u].load(src + (h + u) * x.sh + it.d1);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (h + u >= h1) break;
      float a[8], c[8];
      v[u].floats(a);
      w[u].floats(c);
      if (in) it.turn(a, c, src + (h + u) * x.sh, rt);
      T* o = dst + (long long)(h + u) * Tn * d;
      q8_store8(o + it.d0, a);
      if (MODE == kRotPairs && it.d1 >= 0) q8_store8(o + it.d1, c);
    }
  }
}

// One thread: one item of one token for hpt heads (of q, then k). Bound: HBM, every row read and written once; a token's
// table row (4 rot bytes) is read by heads / hpt threads an item, from L2 after the first. 2 x 8191 tokens of 32 + 8 fp32
// heads, interleaved, 64 of 128 dimensions: 109 us, 6.2 TB/s (a thread a chunk and head, table read each time: 180 us);
// 8192 tokens, bf16, half layout: 32 us, 5.4 TB/s. Half layouts whose rotated width is no multiple of 16 read partners one
// by one: 62 us for the same tokens with 20 dimensions rotated.
template <typename T, int MODE>
__global__ void __launch_bounds__(256) rotary_kernel(const RotaryParams p) {
  const unsigned i = blockIdx.x * 256u + threadIdx.x;
  const unsigned tok = i / (unsigned)p.items;
  if (tok >= (unsigned)p.B * (unsigned)p.T) return;
  const int item = (int)(i - tok * (unsigned)p.items);
  const int b = (int)(tok / (unsigned)p.T), t = (int)(tok - (unsigned)b * (unsigned)p.T);
  const long long pos = p.pos ? p.pos[b * p.pos_sb + t * p.pos_st] : p.start + t;
  const bool in = pos >= 0 && pos < p.rt.rows;
  if (!in && pos >= 0 && item == 0 && blockIdx.y == 0) atomicOr(p.err, kErrQ8Range);
  RotItem<MODE> it;
  it.init(p.rt, p.rt.table + (in ? pos * p.rt.rot : 0), item, p.sgn);
  constexpr int U = sizeof(T) == 2 ? 4 : 2;
  const int h0 = blockIdx.y * p.hpt, h1 = min(h0 + p.hpt, p.q.H + p.k.H);
  if (h0 < p.q.H) rot_heads<T, MODE, U>(p.q, h0, min(h1, p.q.H), b, t, p.T, p.d, it, p.rt, in);
  if (h1 > p.q.H) rot_heads<T, MODE, U>(p.k, max(h0 - p.q.H, 0), h1 - p.q.H, b, t, p.T, p.d, it, p.rt, in);
}

// ------------------------------------------------------------------------------------------------ quantising write
struct Q8AppendParams {
  uint8_t* codes[2];          // K, V [B,G,C,128]
  signed char* exps[2];       // [B,G,NB]
  const void* x[2];           // new rows [B,G,T,128] (strides sb, sg, st)
  long long sb[2], sg[2], st[2];
  Q8Lengths len;
  int B, G, T, C, NB;
  int touched;                // blocks a request's T rows can reach
  RotTable rt;                // rt.table null: no rotation
  RotTensor q;                // queries to rotate, [B, G*h, T, 128] with head (g, i) at g * q_sg + i * sh; x null: none
  long long q_sg;
  int h;
  int items, hpt;             // of q's rotation
  int kv_ctas;                // CTAs of the write; the rest rotate q
  unsigned* err;
};

constexpr int kQ8AppendThreads = 256;      // 8 threads a row, two chunks of 8 dimensions each; 32 rows at a time, twice

// One CTA writes one block (64 tokens) of one (batch, group) of K or V: the new rows are read once into registers,
// rotated (K), their largest finite value reduced over the CTA, then rounded and stored: the block's scale needs no pass
// of its own, because the block is the CTA's tile. Rows the block already holds are touched only when the exponent grows.
// A thread's two chunks are a rotation pair (kRotPairs) or its own columns. Bound: HBM (2 or 4 bytes in, 1 out per
// element; q's rotation reads and writes as much again per head).
template <typename T, int MODE>
__device__ __forceinline__ void q8_append_block(const Q8AppendParams& p, int kv, int bg, int n_idx) {
  __shared__ uint32_t s_max[kQ8AppendThreads / 32];
  const int tid = threadIdx.x, item = tid & 7, r0 = tid >> 3;
  const int b = bg / p.G, g = bg - b * p.G;
  const int len = q8_length(p.len, b), n = min(len, p.C);
  if ((len < 0 || len > p.C) && tid == 0) atomicOr(p.err, kErrQ8Range);
  if (len <= 0 || len - p.T >= p.C) return;
  const int start = len - p.T;                       // position of new row 0 (negative: padded on the left)
  const int blk = max(start, 0) / kQ8Block + n_idx, p0 = blk * kQ8Block;
  if (p0 >= n) return;
  const T* src = static_cast<const T*>(p.x[kv]) + b * p.sb[kv] + g * p.sg[kv];
  const bool turn = kv == 0 && p.rt.table != nullptr;
  // chunks of this thread: the pair of its item where items pair up (rot = 128), else columns 8 item and 64 + 8 item
  const int d0 = 8 * item, d1 = 64 + 8 * item;
  float x[2][8], y[2][8];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int pos = p0 + r0 + 32 * i;
#pragma unroll
    for (int j = 0; j < 8; ++j) x[i][j] = y[i][j] = 0.0f;
    if (pos >= start && pos < n) {
      q8_load8(src + (long long)(pos - start) * p.st[kv] + d0, x[i]);
      q8_load8(src + (long long)(pos - start) * p.st[kv] + d1, y[i]);
    }
  }
  signed char* ep = p.exps[kv] + (long long)bg * p.NB + blk;
  const int kept = min(max(start - p0, 0), kQ8Block);   // rows the block already holds
  const int e_old = kept > 0 ? (int)*ep : kQ8EMin;
  uint32_t amax = 0;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int pos = p0 + r0 + 32 * i;
    if (turn && pos >= start && pos < n) {
      if (pos < p.rt.rows) {
        const float* tr = p.rt.table + (long long)pos * p.rt.rot;
        const T* row = src + (long long)(pos - start) * p.st[0];
        if (MODE == kRotPairs && p.rt.rot == kHeadDim) {
          RotItem<kRotPairs> it;
          it.init(p.rt, tr, item, 1.0f);
          it.turn(x[i], y[i], row, p.rt);
        } else {
          // chunk by chunk; partners outside it come from the row
          constexpr int M = MODE == kRotInner ? kRotInner : kRotOdd;
          RotItem<M> it;
          it.init(p.rt, tr, item, 1.0f);
          it.turn(x[i], y[i], row, p.rt);
          it.init(p.rt, tr, 8 + item, 1.0f);
          it.turn(y[i], x[i], row, p.rt);
        }
      } else {
        if (item == 0) atomicOr(p.err, kErrQ8Range);
#pragma unroll
        for (int j = 0; j < 8; ++j) x[i][j] = y[i][j] = 0.0f;
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (q8_finite(x[i][j])) amax = max(amax, __float_as_uint(x[i][j]) & 0x7fffffffu);
      else x[i][j] = __uint_as_float(0x7fffffffu);
      if (q8_finite(y[i][j])) amax = max(amax, __float_as_uint(y[i][j]) & 0x7fffffffu);
      else y[i][j] = __uint_as_float(0x7fffffffu);
    }
  }
  amax = __reduce_max_sync(0xffffffffu, amax);
  if ((tid & 31) == 0) s_max[tid >> 5] = amax;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kQ8AppendThreads / 32; ++w) amax = max(amax, s_max[w]);
  const int e = max(e_old, q8_exponent(amax));
  const float inv = q8_exp2i(-e);
  uint8_t* dst = p.codes[kv] + ((long long)bg * p.C + p0) * kHeadDim;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = r0 + 32 * i, pos = p0 + r;
    uint2* o0 = reinterpret_cast<uint2*>(dst + r * kHeadDim + d0);
    uint2* o1 = reinterpret_cast<uint2*>(dst + r * kHeadDim + d1);
    if (pos >= start && pos < n) {
      *o0 = q8_encode8(x[i], inv);
      *o1 = q8_encode8(y[i], inv);
    } else if (r < kept && e != e_old) {
      const float shift = q8_exp2i(e_old - e);
      q8_decode8(*o0, x[i]);
      q8_decode8(*o1, y[i]);
      *o0 = q8_encode8(x[i], shift);
      *o1 = q8_encode8(y[i], shift);
    }
  }
  if (tid == 0) *ep = (signed char)e;
}

// Four CTAs an SM for the aligned pairs (with two rows of q in flight a thread): 39.5 us for 8192 tokens of 32/8 heads
// against 47.6 us with four rows in flight and two CTAs; the other layouts hold fewer registers and gain nothing.
template <typename T, int MODE>
__global__ void __launch_bounds__(kQ8AppendThreads, MODE == kRotPairs ? 4 : 2) q8_append_kernel(const Q8AppendParams p) {
  const unsigned blk = blockIdx.x;
  if (blk < (unsigned)p.kv_ctas) {
    // block index fastest, then K / V, then (batch, group)
    const unsigned rest = blk / (unsigned)p.touched;
    q8_append_block<T, MODE>(p, (int)(rest & 1), (int)(rest >> 1), (int)(blk - rest * (unsigned)p.touched));
    return;
  }
  // q: one thread rotates one item of one token for hpt heads of one group
  const unsigned i = (blk - (unsigned)p.kv_ctas) * kQ8AppendThreads + threadIdx.x;
  const unsigned tok = i / (unsigned)p.items;
  const int item = (int)(i - tok * (unsigned)p.items);
  const unsigned split = (unsigned)((p.h + p.hpt - 1) / p.hpt);      // threads over a group's heads
  const unsigned bgs = tok / (unsigned)p.T;
  const int t = (int)(tok - bgs * (unsigned)p.T);
  const unsigned bg = bgs / split;
  if (bg >= (unsigned)(p.B * p.G)) return;
  const int b = (int)(bg / (unsigned)p.G), g = (int)(bg - (unsigned)b * (unsigned)p.G);
  const int h0 = (int)(bgs - bg * split) * p.hpt;
  const long long pos = (long long)q8_length(p.len, b) - p.T + t;
  const bool in = pos >= 0 && pos < p.rt.rows;
  if (!in && pos >= 0 && item == 0) atomicOr(p.err, kErrQ8Range);
  RotItem<MODE> it;
  it.init(p.rt, p.rt.table + (in ? pos * p.rt.rot : 0), item, 1.0f);
  RotTensor x = p.q;                       // this group's heads as a tensor of its own
  x.x = static_cast<const T*>(p.q.x) + b * p.q.sb + g * p.q_sg;
  x.out = static_cast<T*>(p.q.out) + (long long)bg * p.h * p.T * kHeadDim;
  x.sb = 0;
  rot_heads<T, MODE, MODE == kRotPairs || sizeof(T) == 4 ? 2 : 4>(x, h0, min(h0 + p.hpt, p.h), 0, t, p.T, kHeadDim, it, p.rt, in);
}

// ------------------------------------------------------------------------------------------------ read-back
struct Q8ReadParams {
  const uint8_t* codes[2];
  const signed char* exps[2];
  void* out[2];               // [B,G,hi-lo,128] contiguous
  int C, NB, lo, hi;
};

// One CTA reads one block's rows of one (batch, group) of K or V (grid: blocks, B*G, 2), so a CTA has one exponent and
// no divisions. A thread writes 16 bytes at a time (8 bf16 or 4 fp32), so a warp's stores are contiguous; all of its
// loads are in flight together. Bound: HBM, 1 byte in and 2 or 4 out per element. 8 heads of 131072 tokens to bf16:
// 122 us, 6.6 TB/s (one row a thread with 64-bit divisions: 363 us).
template <typename T>
__global__ void __launch_bounds__(256) q8_read_kernel(const Q8ReadParams p) {
  constexpr int E = 16 / (int)sizeof(T);             // elements per thread and row
  constexpr int L = kHeadDim / E, RPT = 256 / L;     // threads per row, rows at a time
  constexpr int N = kQ8Block / RPT;                  // rows per thread
  const int kv = blockIdx.z, blk = p.lo / kQ8Block + (int)blockIdx.x;
  const long long bg = blockIdx.y;
  const int r0 = threadIdx.x / L, c = (threadIdx.x % L) * E;
  const int p0 = blk * kQ8Block + r0;
  const float scale = q8_exp2i((kv ? p.exps[1] : p.exps[0])[bg * p.NB + blk]);
  const uint8_t* src = (kv ? p.codes[1] : p.codes[0]) + (bg * p.C + p0) * kHeadDim + c;
  T* dst = static_cast<T*>(kv ? p.out[1] : p.out[0]) + (bg * (p.hi - p.lo) + (p0 - p.lo)) * kHeadDim + c;
  uint32_t w[N][E / 4];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int pos = p0 + i * RPT;
    if (pos >= p.lo && pos < p.hi) {
      if constexpr (E == 8) {
        const uint2 v = __ldg(reinterpret_cast<const uint2*>(src + i * RPT * kHeadDim));
        w[i][0] = v.x;
        w[i][1] = v.y;
      } else {
        w[i][0] = __ldg(reinterpret_cast<const uint32_t*>(src + i * RPT * kHeadDim));
      }
    }
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int pos = p0 + i * RPT;
    if (pos < p.lo || pos >= p.hi) continue;
    float f[E];
#pragma unroll
    for (int j = 0; j < E / 4; ++j) {
      const float2 a = q8_half2_floats(q8_decode_lo(w[i][j])), b = q8_half2_floats(q8_decode_hi(w[i][j]));
      f[4 * j] = a.x * scale; f[4 * j + 1] = a.y * scale; f[4 * j + 2] = b.x * scale; f[4 * j + 3] = b.y * scale;
    }
    uint4 o;
    if constexpr (E == 8)
      o = make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
    else
      o = make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
    *reinterpret_cast<uint4*>(dst + i * RPT * kHeadDim) = o;
  }
}

}  // namespace al
