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

// 8 elements of T as floats.
__device__ __forceinline__ void q8_load8(const __nv_bfloat16* p, float (&f)[8]) {
  unpack(*reinterpret_cast<const uint4*>(p), f, p);
}
__device__ __forceinline__ void q8_load8(const float* p, float (&f)[8]) {
  unpack(reinterpret_cast<const uint4*>(p)[0], f, p);
  unpack(reinterpret_cast<const uint4*>(p)[1], f + 4, p);
}
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

// Rotate the 8 dimensions [8 ch, 8 ch + 8) of the row at `row` (held in x); partners outside the chunk are read from
// the row (it was just read by a neighbouring lane, so these reads hit L1). tr: the position's table row.
template <typename T>
__device__ __forceinline__ void rot_chunk(float (&x)[8], const T* row, const float* tr, int ch, const RotTable& rt,
                                          float sgn) {
  const int half = rt.rot >> 1, d0 = 8 * ch;
  if (d0 >= rt.rot) return;
  if (rt.layout == kRotInterleaved) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int pi = (d0 >> 1) + i;
      if (pi < half) rot_pair(x[2 * i], x[2 * i + 1], __ldg(tr + pi), sgn * __ldg(tr + half + pi));
    }
  } else if ((half & 7) == 0) {
    const bool low = d0 < half;
    const int i0 = low ? d0 : d0 - half;
    float y[8];
    q8_load8(row + (low ? d0 + half : d0 - half), y);
    const float4 c0 = __ldg(reinterpret_cast<const float4*>(tr + i0)), c1 = __ldg(reinterpret_cast<const float4*>(tr + i0) + 1);
    const float4 s0 = __ldg(reinterpret_cast<const float4*>(tr + half + i0)),
                 s1 = __ldg(reinterpret_cast<const float4*>(tr + half + i0) + 1);
    const float c[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w};
    const float s[8] = {s0.x, s0.y, s0.z, s0.w, s1.x, s1.y, s1.z, s1.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float si = sgn * s[i];
      x[i] = low ? __fsub_rn(__fmul_rn(x[i], c[i]), __fmul_rn(y[i], si))
                 : __fadd_rn(__fmul_rn(x[i], c[i]), __fmul_rn(y[i], si));
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int d = d0 + i;
      if (d >= rt.rot) continue;
      const bool low = d < half;
      const int pi = low ? d : d - half;
      const float y = tof(row[low ? d + half : d - half]);
      const float c = __ldg(tr + pi), si = sgn * __ldg(tr + half + pi);
      x[i] = low ? __fsub_rn(__fmul_rn(x[i], c), __fmul_rn(y, si)) : __fadd_rn(__fmul_rn(x[i], c), __fmul_rn(y, si));
    }
  }
}

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
  int hpt;                    // heads per thread
  float sgn;                  // -1: the inverse rotation (the gradient)
  unsigned* err;
};

// One thread: 8 dimensions of one token for hpt heads (of q, then k).
template <typename T>
__global__ void __launch_bounds__(256) rotary_kernel(const RotaryParams p) {
  const int chunks = p.d >> 3;
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  const long long tok = i / chunks;
  if (tok >= (long long)p.B * p.T) return;
  const int ch = (int)(i - tok * chunks);
  const int b = (int)(tok / p.T), t = (int)(tok - (long long)b * p.T);
  const long long pos = p.pos ? p.pos[b * p.pos_sb + t * p.pos_st] : p.start + t;
  const bool in = pos >= 0 && pos < p.rt.rows;
  if (!in && pos >= 0 && ch == 0 && blockIdx.y == 0) atomicOr(p.err, kErrQ8Range);
  const float* tr = p.rt.table + (in ? pos * p.rt.rot : 0);
  const int h0 = blockIdx.y * p.hpt, h1 = min(h0 + p.hpt, p.q.H + p.k.H);
  for (int hh = h0; hh < h1; ++hh) {
    const bool second = hh >= p.q.H;
    const RotTensor& x = second ? p.k : p.q;
    const int head = second ? hh - p.q.H : hh;
    const T* row = static_cast<const T*>(x.x) + b * x.sb + head * x.sh + t * x.st;
    float v[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    if (in) {
      q8_load8(row + 8 * ch, v);
      rot_chunk(v, row, tr, ch, p.rt, p.sgn);
    }
    q8_store8(static_cast<T*>(x.out) + (((long long)b * x.H + head) * p.T + t) * p.d + 8 * ch, v);
  }
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
  const void* q;              // queries to rotate [B,G,h,T,128] (strides) or null
  long long q_sb, q_sg, q_sh, q_st;
  int h;
  void* q_out;                // contiguous [B,G,h,T,128]
  int kv_ctas;                // CTAs of the write; the rest rotate q
  unsigned* err;
};

constexpr int kQ8AppendThreads = 128;      // 16 lanes x 8 dimensions per row, 8 rows at a time, 8 times

// One CTA writes one block (64 tokens) of one (batch, group) of K or V: the new rows are read once into registers,
// rotated (K), their largest finite value reduced over the CTA, then rounded and stored. Rows the block already holds
// are touched only when the exponent grows.
template <typename T>
__device__ __forceinline__ void q8_append_block(const Q8AppendParams& p, int kv, int bg, int n_idx) {
  __shared__ uint32_t s_max[kQ8AppendThreads / 32];
  const int tid = threadIdx.x, ch = tid & 15, r0 = tid >> 4;
  const int b = bg / p.G, g = bg - b * p.G;
  const int len = q8_length(p.len, b), n = min(len, p.C);
  if ((len < 0 || len > p.C) && tid == 0) atomicOr(p.err, kErrQ8Range);
  if (len <= 0 || len - p.T >= p.C) return;
  const int start = len - p.T;                       // position of new row 0 (negative: padded on the left)
  const int blk = max(start, 0) / kQ8Block + n_idx, p0 = blk * kQ8Block;
  if (p0 >= n) return;
  const T* src = static_cast<const T*>(p.x[kv]) + b * p.sb[kv] + g * p.sg[kv];
  const bool turn = kv == 0 && p.rt.table != nullptr;
  float x[8][8];
  uint32_t amax = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int pos = p0 + r0 + 8 * i;
    const bool fresh = pos >= start && pos < n;
#pragma unroll
    for (int j = 0; j < 8; ++j) x[i][j] = 0.0f;
    if (fresh) q8_load8(src + (long long)(pos - start) * p.st[kv] + 8 * ch, x[i]);
  }
  if (turn) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int pos = p0 + r0 + 8 * i;
      if (pos < start || pos >= n) continue;
      if (pos < p.rt.rows) {
        rot_chunk(x[i], src + (long long)(pos - start) * p.st[0], p.rt.table + (long long)pos * p.rt.rot, ch, p.rt, 1.0f);
      } else {
        if (ch == 0) atomicOr(p.err, kErrQ8Range);
#pragma unroll
        for (int j = 0; j < 8; ++j) x[i][j] = 0.0f;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (q8_finite(x[i][j])) amax = max(amax, __float_as_uint(x[i][j]) & 0x7fffffffu);
      else x[i][j] = __uint_as_float(0x7fffffffu);
    }
  amax = __reduce_max_sync(0xffffffffu, amax);
  if ((tid & 31) == 0) s_max[tid >> 5] = amax;
  signed char* ep = p.exps[kv] + (long long)bg * p.NB + blk;
  const int kept = min(max(start - p0, 0), kQ8Block);   // rows the block already holds
  const int e_old = kept > 0 ? (int)*ep : kQ8EMin;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kQ8AppendThreads / 32; ++w) amax = max(amax, s_max[w]);
  const int e = max(e_old, q8_exponent(amax));
  const float inv = q8_exp2i(-e);
  uint8_t* dst = p.codes[kv] + ((long long)bg * p.C + p0) * kHeadDim + 8 * ch;
  const float shift = q8_exp2i(e_old - e);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = r0 + 8 * i, pos = p0 + r;
    uint2* out = reinterpret_cast<uint2*>(dst + r * kHeadDim);
    if (pos >= start && pos < n) {
      float y[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] = __fmul_rn(x[i][j], inv);
      *out = make_uint2(q8_encode2(y[0], y[1]) | (q8_encode2(y[2], y[3]) << 16),
                        q8_encode2(y[4], y[5]) | (q8_encode2(y[6], y[7]) << 16));
    } else if (r < kept && e != e_old) {
      uint2 w = *out;
      const float2 a = q8_half2_floats(q8_decode_lo(w.x)), c = q8_half2_floats(q8_decode_hi(w.x));
      const float2 f = q8_half2_floats(q8_decode_lo(w.y)), u = q8_half2_floats(q8_decode_hi(w.y));
      w.x = q8_encode2(a.x * shift, a.y * shift) | (q8_encode2(c.x * shift, c.y * shift) << 16);
      w.y = q8_encode2(f.x * shift, f.y * shift) | (q8_encode2(u.x * shift, u.y * shift) << 16);
      *out = w;
    }
  }
  if (tid == 0) *ep = (signed char)e;
}

template <typename T>
__global__ void __launch_bounds__(kQ8AppendThreads) q8_append_kernel(const Q8AppendParams p) {
  const long long blk = blockIdx.x;
  if (blk < p.kv_ctas) {
    // block index fastest, then K / V, then (batch, group)
    const int n_idx = (int)(blk % p.touched);
    const long long rest = blk / p.touched;
    q8_append_block<T>(p, (int)(rest & 1), (int)(rest >> 1), n_idx);
    return;
  }
  // q: one thread rotates 8 dimensions of one (b, g, head, t) row
  const long long i = (blk - p.kv_ctas) * kQ8AppendThreads + threadIdx.x;
  const long long row = i >> 4;
  const int ch = (int)(i & 15);
  const int per_b = p.G * p.h * p.T;
  if (row >= (long long)p.B * per_b) return;
  const int b = (int)(row / per_b);
  int rem = (int)(row - (long long)b * per_b);
  const int t = rem % p.T;
  rem /= p.T;
  const int head = rem % p.h, g = rem / p.h;
  const long long pos = (long long)q8_length(p.len, b) - p.T + t;
  const bool in = pos >= 0 && pos < p.rt.rows;
  if (!in && pos >= 0 && ch == 0) atomicOr(p.err, kErrQ8Range);
  const T* src = static_cast<const T*>(p.q) + b * p.q_sb + g * p.q_sg + head * p.q_sh + t * p.q_st;
  float v[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
  if (in) {
    q8_load8(src + 8 * ch, v);
    rot_chunk(v, src, p.rt.table + pos * p.rt.rot, ch, p.rt, 1.0f);
  }
  q8_store8(static_cast<T*>(p.q_out) + row * kHeadDim + 8 * ch, v);
}

// ------------------------------------------------------------------------------------------------ read-back
struct Q8ReadParams {
  const uint8_t* codes[2];
  const signed char* exps[2];
  void* out[2];               // [B,G,hi-lo,128] contiguous
  int C, NB, lo, n;           // n = hi - lo
  long long rows;             // B*G*n
};

// One thread: 16 bytes of output (8 bf16 or 4 fp32), so that a warp's stores are contiguous.
template <typename T>
__global__ void __launch_bounds__(256) q8_read_kernel(const Q8ReadParams p) {
  constexpr int E = 16 / (int)sizeof(T);             // elements per thread
  constexpr int L = kHeadDim / E;                    // threads per row
  const int kv = blockIdx.y;
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  const long long row = i / L;
  if (row >= p.rows) return;
  const int c = (int)(i % L) * E;
  const long long bg = row / p.n;
  const int pos = p.lo + (int)(row - bg * p.n);
  const float scale = q8_exp2i(p.exps[kv][bg * p.NB + pos / kQ8Block]);
  const uint8_t* src = p.codes[kv] + (bg * p.C + pos) * kHeadDim + c;
  T* dst = static_cast<T*>(p.out[kv]) + row * kHeadDim + c;
  uint32_t w[E / 4];
  if (E == 8) {
    const uint2 v = __ldg(reinterpret_cast<const uint2*>(src));
    w[0] = v.x;
    w[E / 4 - 1] = v.y;
  } else {
    w[0] = __ldg(reinterpret_cast<const uint32_t*>(src));
  }
  float f[E];
#pragma unroll
  for (int j = 0; j < E / 4; ++j) {
    const float2 a = q8_half2_floats(q8_decode_lo(w[j])), b = q8_half2_floats(q8_decode_hi(w[j]));
    f[4 * j] = a.x * scale; f[4 * j + 1] = a.y * scale; f[4 * j + 2] = b.x * scale; f[4 * j + 3] = b.y * scale;
  }
  if (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(dst) = make_float4(f[0], f[1], f[2], f[3]);
  } else {
    *reinterpret_cast<uint4*>(dst) = make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]),
                                                pack_bf16x2(f[E - 4], f[E - 3]), pack_bf16x2(f[E - 2], f[E - 1]));
  }
}

}  // namespace al
