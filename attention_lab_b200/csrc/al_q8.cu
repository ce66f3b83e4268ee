// C ABI of the 8-bit cache: validation, launch-shape choice and dispatch.
// Declarations and contracts: include/attention_lab_b200.h.
#include <algorithm>

#include "al_host.h"
#include "al_q8_prompt.cuh"

using namespace al;

namespace {

bool rows_aligned(const void* p, int dtype, int64_t s0, int64_t s1, int64_t s2, int64_t s3 = 0) {
  return aligned16(p) && ((s0 | s1 | s2 | s3) & (16 / esize(dtype) - 1)) == 0;
}

int rot_table(const float* table, int rows, int rot, int layout, int d, RotTable* out) {
  if (!table) return fail(AL_EINVAL, "null rotary table");
  if (rows < 1) return fail(AL_EINVAL, "the rotary table needs at least one row");
  if (rot < 2 || rot % 2 || rot > d) return fail(AL_EINVAL, "rotary_dim must be even and in [2, head_dim=%d], got %d", d, rot);
  if (layout != AL_ROT_HALF && layout != AL_ROT_INTERLEAVED) return fail(AL_EINVAL, "unknown rotary layout %d", layout);
  if (!aligned16(table)) return fail(AL_EUNSUPPORTED, "the rotary table must start on a 16-byte boundary");
  out->table = table; out->rows = rows; out->rot = rot; out->layout = layout;
  return AL_OK;
}

// Shape checks every 8-bit cache entry shares.
int q8_shape(int B, int G, int C, int d, const void* kc, const void* vc, const void* ke, const void* ve) {
  if (B < 0 || G <= 0 || C <= 0) return fail(AL_EINVAL, "G and C must be positive and B not negative");
  if (d != kHeadDim) return fail(AL_EUNSUPPORTED, "head_dim must be %d, got %d", kHeadDim, d);
  if (B * (long long)G > 65535) return fail(AL_EUNSUPPORTED, "B*G = %lld exceeds 65535", B * (long long)G);
  if (B == 0) return AL_OK;
  if (!kc || !vc || !ke || !ve) return fail(AL_EINVAL, "null cache pointer");
  if (!aligned16(kc) || !aligned16(vc)) return fail(AL_EUNSUPPORTED, "the codes must start on a 16-byte boundary");
  return AL_OK;
}

int q8_blocks(int C) { return (C - 1) / kQ8Block + 1; }

template <typename T>
void rotary_launch(int mode, dim3 grid, cudaStream_t st, const RotaryParams& p) {
  if (mode == kRotPairs) rotary_kernel<T, kRotPairs><<<grid, 256, 0, st>>>(p);
  else if (mode == kRotInner) rotary_kernel<T, kRotInner><<<grid, 256, 0, st>>>(p);
  else rotary_kernel<T, kRotOdd><<<grid, 256, 0, st>>>(p);
}
template <typename T>
void append_launch(int mode, unsigned grid, cudaStream_t st, const Q8AppendParams& p) {
  if (mode == kRotPairs) q8_append_kernel<T, kRotPairs><<<grid, kQ8AppendThreads, 0, st>>>(p);
  else if (mode == kRotInner) q8_append_kernel<T, kRotInner><<<grid, kQ8AppendThreads, 0, st>>>(p);
  else q8_append_kernel<T, kRotOdd><<<grid, kQ8AppendThreads, 0, st>>>(p);
}

// The attend's kernel, and how it splits its work.
struct Q8Plan {
  bool token;                       // the few-column kernel (mma.sync); else the prompt kernel (tcgen05)
  int cs, chunk;                    // token: CTAs per cluster; steps per CTA of a split
  int row_tiles, tile_rows;         // prompt: CTAs along a group's query rows, rows a CTA (128 or 256)
  int nsplit;                       // key splits merged through the workspace
  size_t ml_off, bytes;             // nsplit > 1: workspace layout
};

int q8_plan(int B, int G, int h, int T, int C, int window, int sinks, int max_length, bool ragged, bool wide, int sms, Q8Plan* out) {
  Q8Plan pl = {};
  pl.nsplit = 1;
  const long long R = (long long)h * T, segs = (long long)B * G;
  int len = max_length > 0 ? std::min(max_length, C) : C;
  // tokens a query tile can see, as far as the host knows
  const long long span = window > 0 ? std::min<long long>(len, (long long)window + sinks) : len;
  // (Times in this function: graph replays in bursts at the full clock, 1965 MHz; longer runs of the large ones are 10 to
  // 15 % slower under the power cap.)
  // The few-column kernel reads the cache once per 8 query rows, the prompt kernel once per 256 but fills 128 x 128 tiles
  // and takes 8 us for the least work. Up to 16 rows the first wins throughout (16 heads over 32 x 8192 tokens: 175 us
  // against 211); up to 128 while everything it reads is small (one request, 8 groups: 64 rows over 512 tokens 5.8 us
  // against 13.6, over 4096 tokens 15.4 against 15.1; 32 rows over 32 x 8192 tokens 317 against 215).
  const long long ngrp = (R + kQdCols - 1) / kQdCols, units = segs * ngrp;
  if (R <= kQ8TokenCols || (R <= kQ8FewCols && units * span <= kQ8FewTokens)) {
    pl.token = true;
    // One wave: clusters grow while the CTAs (two an SM) still fit at once and every warp keeps a step (two before the
    // first doubling, which brings the exchange). 8 segments of 2048 tokens: 8 CTAs each 5.4 us, 16 5.2; 128 of 256
    // tokens: one CTA each 4.9, two 5.8.
    pl.cs = 1;
    while (pl.cs < kMaxCluster && units * pl.cs * 2 <= 2LL * sms && span >= pl.cs * (pl.cs == 1 ? 4LL : 2LL) * kQdWarps * kQdStep)
      pl.cs <<= 1;
    // Splits merged by a second kernel: more CTAs a segment than clusters spread over the SMs (one request of 128K: 48 us
    // against 89; 6 x 8 segments of 4100 tokens: 13.8 against 16.4), and for requests of their own lengths runs of 4096
    // tokens, so that the load evens out whatever the lengths are: 256 segments of 16K to 32K tokens 259 us against 316
    // with clusters, 64 of 100 to 32K 54 against 72; 64 segments that all have 32K lose, 97 against 91.
    long long fill = std::min<long long>(2LL * sms / units, span / (2 * kQdWarps * kQdStep));
    if (ragged) fill = std::max<long long>(fill, span / kQdChunk);
    fill = std::min<long long>(fill, 32 * kQmWarps);
    if (fill >= 3 && fill > pl.cs) {
      const long long steps = span / kQdStep + 2;
      pl.cs = 1;
      pl.chunk = (int)((steps + fill - 1) / fill);
      pl.nsplit = (int)((steps + pl.chunk - 1) / pl.chunk);
    }
  } else {
    // A CTA takes 128 or 256 query rows (32-bit queries 128), and with few CTAs the keys are split and the splits merged. What a call's time
    // measured as, in tenths of a microsecond for bf16 (fp32: all about 1.4 times that): 70 and 16 a key tile with 128
    // rows, 80 and 21 with 256, 50 for the splits' partial results and their merge; the least is taken. 32/8 heads: a
    // prompt of 512 tokens 14.9 us (128 rows; 256 rows, keys split, 20.4), 64 rows late in 2048 tokens 15.3 (128 rows in
    // 8 splits; 256 rows in 4, 20.8), 256 tokens late in 4096 34.5 (256 rows in 4 splits; 128 rows in 2, 41.6).
    long long best = 0;
    for (int rows = kQpRows; rows <= 2 * kQpRows; rows += kQpRows) {
      const long long ctas = segs * ((R + rows - 1) / rows);
      if (wide ? rows > kQpRows : rows == kQpRows && ctas > sms) continue;   // 32-bit queries: always 128 (kQpFlush)
      const long long seen = window > 0 ? std::min<long long>(len, (long long)window + sinks + rows / h + kQpKeys) : len;
      const long long tiles = (seen + kQpKeys - 1) / kQpKeys, most = std::max<long long>(1, std::min<long long>(sms / ctas, tiles / 2));
      for (long long ns = 1; ns <= most; ns += std::max<long long>(1, most - 1)) {
        const long long t = (tiles + ns - 1) / ns, cost = (rows == kQpRows ? 70 + 16 * t : 80 + 21 * t) + (ns > 1 ? 50 : 0);
        if (best > 0 && cost >= best) continue;
        best = cost;
        pl.tile_rows = rows;
        pl.row_tiles = (int)((R + rows - 1) / rows);
        pl.nsplit = (int)ns;
      }
    }
  }
  if (pl.nsplit > 1) {
    const size_t rows = (size_t)segs * (size_t)R;
    pl.ml_off = (size_t)pl.nsplit * rows * kHeadDim * sizeof(float);
    pl.bytes = pl.ml_off + (size_t)pl.nsplit * rows * 2 * sizeof(float);
  }
  *out = pl;
  return AL_OK;
}

// A window or sinks as large as the cache hide nothing, and are passed on as none: the kernels subtract the window from
// positions down to -T (at least -2^25, below) in 32 bits, which holds for a window smaller than a cache that fits memory.
void q8_visible(int C, int* window, int* sinks) {
  if (*window >= C || *sinks >= C) *window = 0;
  if (*window == 0) *sinks = 0;
}

int q8_attend_check(int B, int G, int h, int T, int window, int sinks) {
  if (h < 1 || T < 0) return fail(AL_EINVAL, "h must be positive and T not negative, got h=%d T=%d", h, T);
  if (window < 0 || sinks < 0) return fail(AL_EINVAL, "window and sinks must not be negative, got %d and %d", window, sinks);
  if (h > 64) return fail(AL_EUNSUPPORTED, "heads per group must be in [1, 64], got %d", h);
  if ((long long)h * T > (1 << 25)) return fail(AL_EUNSUPPORTED, "h*T = %lld exceeds 2^25 query rows per group", (long long)h * T);
  if (B * (long long)G * (((long long)h * T + 255) / 256) > 0x7fffffffLL) return fail(AL_EUNSUPPORTED, "too many query tiles");
  if (B * (long long)G * h * T > 0x7fffffffLL) return fail(AL_EUNSUPPORTED, "too many query rows");
  return AL_OK;
}

template <typename T>
int q8_launch_attend(const Q8AttendParams& p, const Q8Plan& pl, void* stream) {
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const long long R = (long long)p.h * p.T;
  int rc;
  if (pl.token) {
    if ((rc = prepare_kernel(q8_decode_kernel<T>, kQdSmemOf<T>))) return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(kQdThreads, 1, 1);
    cfg.dynamicSmemBytes = kQdSmemOf<T>;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    cfg.attrs = attr;
    auto shape = [&](int cs) {                         // any power of two will do: the CTAs of a cluster interleave
      cfg.gridDim = dim3((unsigned)(pl.nsplit > 1 ? pl.nsplit : cs), (unsigned)(p.B * p.G), (unsigned)((R + kQdCols - 1) / kQdCols));
      attr[0].val.clusterDim = {(unsigned)cs, 1, 1};
      cfg.numAttrs = cs > 1 ? 1 : 0;
    };
    int cs = 1;
    if ((rc = fitting_cluster(pl.cs, [&](int n, bool* ok) {
           shape(n);
           return cluster_schedulable(reinterpret_cast<const void*>(q8_decode_kernel<T>), cfg, n, ok);
         }, &cs))) return rc;
    shape(cs);
    const cudaError_t e = cudaLaunchKernelEx(&cfg, q8_decode_kernel<T>, p);
    if (e != cudaSuccess) return cuda_fail(e, "q8_decode_kernel");
  } else {
    auto kernel = q8_prompt_kernel<T, 1>;
    if constexpr (sizeof(T) == 2) {
      if (pl.tile_rows > kQpRows) kernel = q8_prompt_kernel<T, 2>;
    }
    if ((rc = prepare_kernel(kernel, kQpSmem))) return rc;
    const dim3 grid((unsigned)(p.B * p.G * pl.row_tiles), (unsigned)pl.nsplit);
    kernel<<<grid, kQpThreads, kQpSmem, st>>>(p);
    if ((rc = plain_launch_check("q8_prompt_kernel"))) return rc;
  }
  if (pl.nsplit > 1) {
    cudaLaunchConfig_t cfg = {};
    const long long rows = (long long)p.B * p.G * R;
    // warps per row: 8 for many splits of few rows, or 1 (18 splits of 2048 rows: 33.2 us in all against 37.8)
    const bool wide = pl.nsplit > 32 || (pl.nsplit > 8 && rows <= 1024);
    cfg.gridDim = dim3((unsigned)(wide ? rows : (rows + kQmWarps - 1) / kQmWarps), 1, 1);
    cfg.blockDim = dim3(32 * kQmWarps, 1, 1);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = wide ? cudaLaunchKernelEx(&cfg, q8_merge_kernel<T, kQmWarps>, p)
                               : cudaLaunchKernelEx(&cfg, q8_merge_kernel<T, 1>, p);
    if (e != cudaSuccess) return cuda_fail(e, "q8_merge_kernel");
  }
  return AL_OK;
}

}  // namespace

extern "C" {

int al_rotary(const void* q, int64_t q_sb, int64_t q_sh, int64_t q_st, int Hq,
              const void* k, int64_t k_sb, int64_t k_sh, int64_t k_st, int Hk, int dtype,
              const float* table, int table_rows, int rot, int layout,
              const int64_t* positions, int64_t pos_sb, int64_t pos_st, int64_t start,
              int B, int T, int d, int inverse, void* q_out, void* k_out, void* stream) {
  if (!dtype_ok(dtype)) return fail(AL_EINVAL, "unknown dtype code");
  if (B < 0 || T < 0 || Hq < 1 || Hk < 0) return fail(AL_EINVAL, "need B, T >= 0, Hq >= 1 and Hk >= 0");
  if (d < 8 || d % 8 || d > 1024) return fail(AL_EUNSUPPORTED, "head_dim must be a multiple of 8 in [8, 1024], got %d", d);
  RotaryParams p = {};
  int rc = rot_table(table, table_rows, rot, layout, d, &p.rt);
  if (rc) return rc;
  if (B == 0 || T == 0) return AL_OK;
  if (!q || !q_out || (Hk > 0 && (!k || !k_out))) return fail(AL_EINVAL, "null pointer argument");
  if (!rows_aligned(q, dtype, q_sb, q_sh, q_st) || !aligned16(q_out) ||
      (Hk > 0 && (!rows_aligned(k, dtype, k_sb, k_sh, k_st) || !aligned16(k_out))))
    return fail(AL_EUNSUPPORTED, "rows must start on 16-byte boundaries");
  DeviceInfo* di = nullptr;
  if ((rc = device_info(&di))) return rc;
  p.q.x = q; p.q.sb = q_sb; p.q.sh = q_sh; p.q.st = q_st; p.q.H = Hq; p.q.out = q_out;
  if (Hk > 0) { p.k.x = k; p.k.sb = k_sb; p.k.sh = k_sh; p.k.st = k_st; p.k.H = Hk; p.k.out = k_out; }
  if (positions) {
    p.pos = reinterpret_cast<const long long*>(positions);
    p.pos_sb = pos_sb; p.pos_st = pos_st;
  }
  p.start = start; p.B = B; p.T = T; p.d = d; p.sgn = inverse ? -1.0f : 1.0f; p.err = di->err;
  const int mode = rot_mode(rot, layout);
  p.items = rot_items(d, rot, mode);
  const long long threads = (long long)B * T * p.items, heads = Hq + Hk;
  const long long blocks = (threads + 255) / 256;
  if (threads > 0x7fffff00LL) return fail(AL_EUNSUPPORTED, "too many tokens for one call");
  // heads per thread: one while the launch does not fill the GPU, then as many as keep it filled (up to 8)
  p.hpt = 1;
  while (p.hpt < 8 && blocks * ((heads + 2 * p.hpt - 1) / (2 * p.hpt)) >= 8LL * di->sms) p.hpt *= 2;
  const long long gy = (heads + p.hpt - 1) / p.hpt;
  if (gy > 65535) return fail(AL_EUNSUPPORTED, "too many heads for one call");
  const dim3 grid((unsigned)blocks, (unsigned)gy);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == AL_F32) rotary_launch<float>(mode, grid, st, p);
  else rotary_launch<__nv_bfloat16>(mode, grid, st, p);
  return plain_launch_check("rotary_kernel");
}

int al_append_q8(void* k_codes, void* v_codes, void* k_exp, void* v_exp, const int* lengths, int length,
                 const void* k_new, int64_t k_sb, int64_t k_sg, int64_t k_st,
                 const void* v_new, int64_t v_sb, int64_t v_sg, int64_t v_st, int dtype,
                 const float* table, int table_rows, int rot, int layout,
                 const void* q, int64_t q_sb, int64_t q_sg, int64_t q_sh, int64_t q_st, int h, void* q_out,
                 int B, int G, int T, int C, int d, void* stream) {
  if (!dtype_ok(dtype)) return fail(AL_EINVAL, "unknown dtype code");
  int rc = q8_shape(B, G, C, d, k_codes, v_codes, k_exp, v_exp);
  if (rc) return rc;
  if (T < 0) return fail(AL_EINVAL, "T must not be negative, got %d", T);
  if (!lengths && (length < T || length > C))
    return fail(AL_EINVAL, "positions [%d, %d) do not fit capacity %d", length - T, length, C);
  Q8AppendParams p = {};
  if (table || q) {
    if ((rc = rot_table(table, table_rows, rot, layout, d, &p.rt))) return rc;
    if (!lengths && length > table_rows)
      return fail(AL_EINVAL, "positions up to %d exceed the rotary table's %d rows", length - 1, table_rows);
  }
  if (B == 0 || T == 0) return AL_OK;
  if (!k_new || !v_new) return fail(AL_EINVAL, "null pointer argument");
  if (!rows_aligned(k_new, dtype, k_sb, k_sg, k_st) || !rows_aligned(v_new, dtype, v_sb, v_sg, v_st))
    return fail(AL_EUNSUPPORTED, "rows must start on 16-byte boundaries");
  if (q) {
    if (h < 1 || !q_out) return fail(AL_EINVAL, "q given without heads or an output");
    if (!rows_aligned(q, dtype, q_sb, q_sg, q_sh, q_st) || !aligned16(q_out)) return fail(AL_EUNSUPPORTED, "rows must start on 16-byte boundaries");
    if ((long long)G * h * T > 0x7fffffffLL) return fail(AL_EUNSUPPORTED, "too many query rows per request");
  }
  DeviceInfo* di = nullptr;
  if ((rc = device_info(&di))) return rc;
  p.codes[0] = static_cast<uint8_t*>(k_codes); p.codes[1] = static_cast<uint8_t*>(v_codes);
  p.exps[0] = static_cast<signed char*>(k_exp); p.exps[1] = static_cast<signed char*>(v_exp);
  p.x[0] = k_new; p.x[1] = v_new;
  p.sb[0] = k_sb; p.sg[0] = k_sg; p.st[0] = k_st;
  p.sb[1] = v_sb; p.sg[1] = v_sg; p.st[1] = v_st;
  p.len.per_batch = lengths; p.len.all = length;
  p.B = B; p.G = G; p.T = T; p.C = C; p.NB = q8_blocks(C);
  p.touched = (int)std::min<long long>(((long long)T + kQ8Block - 2) / kQ8Block + 1, p.NB);
  p.err = di->err;
  const long long kv = 2LL * B * G * p.touched;
  long long qc = 0;
  const int mode = p.rt.table ? rot_mode(rot, layout) : kRotPairs;
  p.items = rot_items(d, rot, mode);
  if (q) {
    p.q.x = q; p.q.sb = q_sb; p.q_sg = q_sg; p.q.sh = q_sh; p.q.st = q_st; p.q.H = h; p.q.out = q_out;
    p.h = h;
    // heads of a group per thread: one while the launch does not fill the GPU, then up to 4 at once
    const long long per = (long long)B * G * T * p.items;
    p.hpt = 1;
    while (p.hpt < 4 && p.hpt < h && per * ((h + 2 * p.hpt - 1) / (2 * p.hpt)) >= 2048LL * di->sms) p.hpt *= 2;
    const long long threads = per * ((h + p.hpt - 1) / p.hpt);
    if (threads > 0x7fffff00LL) return fail(AL_EUNSUPPORTED, "too many query rows for one call");
    qc = (threads + kQ8AppendThreads - 1) / kQ8AppendThreads;
  }
  if (kv + qc > 0x7fffffffLL) return fail(AL_EUNSUPPORTED, "too many rows for one call");
  p.kv_ctas = (int)kv;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const unsigned grid = (unsigned)(kv + qc);
  if (dtype == AL_F32) append_launch<float>(mode, grid, st, p);
  else append_launch<__nv_bfloat16>(mode, grid, st, p);
  return plain_launch_check("q8_append_kernel");
}

int al_read_q8(const void* k_codes, const void* v_codes, const void* k_exp, const void* v_exp, int B, int G, int C, int d,
               int lo, int hi, int out_dtype, void* k_out, void* v_out, void* stream) {
  if (!dtype_ok(out_dtype)) return fail(AL_EINVAL, "unknown dtype code");
  int rc = q8_shape(B, G, C, d, k_codes, v_codes, k_exp, v_exp);
  if (rc) return rc;
  if (!(0 <= lo && lo <= hi && hi <= C)) return fail(AL_EINVAL, "need 0 <= lo <= hi <= C, got lo=%d hi=%d C=%d", lo, hi, C);
  if (B == 0 || lo == hi) return AL_OK;
  if (!k_out || !v_out) return fail(AL_EINVAL, "null output pointer");
  if (!aligned16(k_out) || !aligned16(v_out)) return fail(AL_EUNSUPPORTED, "outputs must start on 16-byte boundaries");
  Q8ReadParams p = {};
  p.codes[0] = static_cast<const uint8_t*>(k_codes); p.codes[1] = static_cast<const uint8_t*>(v_codes);
  p.exps[0] = static_cast<const signed char*>(k_exp); p.exps[1] = static_cast<const signed char*>(v_exp);
  p.out[0] = k_out; p.out[1] = v_out;
  p.C = C; p.NB = q8_blocks(C); p.lo = lo; p.hi = hi;
  const dim3 grid((unsigned)((hi - 1) / kQ8Block - lo / kQ8Block + 1), (unsigned)(B * G), 2);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (out_dtype == AL_F32) q8_read_kernel<float><<<grid, 256, 0, st>>>(p);
  else q8_read_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(p);
  return plain_launch_check("q8_read_kernel");
}

int al_attend_q8_workspace(int B, int G, int h, int T, int C, int window, int sinks, int max_length, size_t* bytes) {
  if (!bytes) return fail(AL_EINVAL, "null bytes");
  *bytes = 0;
  if (B < 0 || G <= 0 || C <= 0) return fail(AL_EINVAL, "G and C must be positive and B not negative");
  int rc = q8_attend_check(B, G, h, T, window, sinks);
  if (rc) return rc;
  q8_visible(C, &window, &sinks);
  if (B == 0 || T == 0) return AL_OK;
  DeviceInfo* di = nullptr;
  if ((rc = device_info(&di))) return rc;
  Q8Plan pl, pl32;
  if ((rc = q8_plan(B, G, h, T, C, window, sinks, max_length, true, false, di->sms, &pl))) return rc;
  if ((rc = q8_plan(B, G, h, T, C, window, sinks, max_length, true, true, di->sms, &pl32))) return rc;
  *bytes = std::max(pl.bytes, pl32.bytes);               // enough for either type
  return AL_OK;
}

int al_attend_q8(const void* q, int64_t q_sb, int64_t q_sg, int64_t q_sh, int64_t q_st, int dtype,
                 const void* k_codes, const void* v_codes, const void* k_exp, const void* v_exp,
                 const int* lengths, int length, int B, int G, int h, int T, int C, int d, int window, int sinks,
                 float scale, int max_length, void* out, void* workspace, size_t workspace_bytes, void* stream) {
  if (!dtype_ok(dtype)) return fail(AL_EINVAL, "unknown dtype code");
  int rc = q8_shape(B, G, C, d, k_codes, v_codes, k_exp, v_exp);
  if (rc) return rc;
  if ((rc = q8_attend_check(B, G, h, T, window, sinks))) return rc;
  q8_visible(C, &window, &sinks);
  if (!lengths && (length < 0 || length > C)) return fail(AL_EINVAL, "length=%d must be in [0, capacity=%d]", length, C);
  if (!(scale == scale) || scale > 3.0e38f || scale < -3.0e38f) return fail(AL_EINVAL, "scale must be finite");
  if (B == 0 || T == 0) return AL_OK;
  if (!q || !out) return fail(AL_EINVAL, "null pointer argument");
  if (!rows_aligned(q, dtype, q_sb, q_sg, q_sh, q_st) || !aligned16(out)) return fail(AL_EUNSUPPORTED, "rows must start on 16-byte boundaries");
  DeviceInfo* di = nullptr;
  if ((rc = device_info(&di))) return rc;
  Q8Plan pl;
  if ((rc = q8_plan(B, G, h, T, C, window, sinks, max_length, lengths != nullptr, dtype == AL_F32, di->sms, &pl))) return rc;
  if (pl.bytes > 0 && (!workspace || workspace_bytes < pl.bytes || !aligned16(workspace)))
    return fail(AL_EINVAL, "this call needs a 16-byte aligned workspace of %zu bytes, got %zu", pl.bytes, workspace_bytes);
  Q8AttendParams p = {};
  p.q = q; p.q_sb = q_sb; p.q_sg = q_sg; p.q_sh = q_sh; p.q_st = q_st;
  p.kc = static_cast<const uint8_t*>(k_codes); p.vc = static_cast<const uint8_t*>(v_codes);
  p.ke = static_cast<const signed char*>(k_exp); p.ve = static_cast<const signed char*>(v_exp);
  p.len.per_batch = lengths; p.len.all = length;
  p.B = B; p.G = G; p.h = h; p.T = T; p.C = C; p.NB = q8_blocks(C);
  p.window = window; p.sinks = sinks;
  p.scale = (scale < 0 ? -scale : scale) * 1.4426950408889634f;
  p.qsign = scale < 0 ? -1.0f : 1.0f;
  p.out = out; p.nsplit = pl.nsplit; p.row_tiles = pl.row_tiles; p.chunk = pl.chunk; p.err = di->err;
  p.h_magic = h > 1 ? 0xffffffffu / (unsigned)h + 1u : 0u;   // exact for r < 2^25, h <= 64: r * (h_magic * h - 2^32) < 2^32
  if (pl.bytes > 0) {
    p.part = static_cast<float*>(workspace);
    p.part_ml = reinterpret_cast<float*>(static_cast<char*>(workspace) + pl.ml_off);
  }
  return dtype == AL_F32 ? q8_launch_attend<float>(p, pl, stream) : q8_launch_attend<__nv_bfloat16>(p, pl, stream);
}

}  // extern "C"
