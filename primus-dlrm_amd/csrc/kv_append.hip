// New keys and values into the pages of an 8-bit cache, keys normed and rotated on the way.
//
// Codes are e4m3, [pages][heads][page_size][D] for keys and for values, with one fp32 scale 2^e per (page,
// head).  Of the values x that a call puts on a page, e is the smallest exponent with max|x| <= 448 * 2^e,
// and at least the page's exponent where the page already holds tokens of the sequence; those are then
// brought to the new scale.  Powers of two cost a floating-point code no precision: code = rne(x * 2^-e) has
// the relative error it would have under any scale, and a rescaled code is exact until it becomes subnormal,
// so a page filled token by token ends up as one filled at once, but for values 2^-14 below its largest.
//
// Bound by HBM (2 bytes read and 1 written per bf16 element) for prompts, by latency for single tokens.  A page's share of
// the batch stays in registers from its load to its codes, so that the maximum costs no second read: 17,800 tokens of 5 prompts,
// 8 heads of 128, 33 us (3.3 TB/s; 49 with keys in one pass and values in another), 1 to 60 tokens of 512 sequences, 6 heads of
// 64, 15.8 us, 64 single tokens behind 100 to 2,000 5.2 us.
#include "kv_common.h"

namespace pdm {
namespace {

struct AppendArgs {
  const void* x[2];           // new keys, new values: element (t, h, d) at t * stride_t + h * stride_h + d
  int64_t stride_t[2], stride_h[2];
  uint8_t* codes[2];
  float* scale[2];
  const int32_t *cu, *table, *lens;
  const void* positions;      // null: the token's index in its sequence
  const float *cos, *sin, *w;
  int32_t* err;
  int64_t tokens, table_stride, table_rows, num_pages;
  int32_t seqs, heads, D, R, page_log2, table_width, bits, width_log2;
  float eps;
};

// Where one page's share of a call's tokens lies.
struct Segment {
  int64_t row0;          // token row of its first token
  int64_t index0;        // that token's index in the sequence
  const int32_t* entry;  // its page
  int slot0, n;          // first slot and number of tokens
};

// The j-th page that sequence b's new tokens touch.
__device__ __forceinline__ bool segment_of(const AppendArgs& a, int b, int64_t c0, int64_t j, Segment& g) {
  const int lg = a.page_log2;
  const int64_t c1 = a.cu[b + 1], len = a.lens[b];
  const int64_t n = c1 - c0;
  if (j < 0 || n <= 0) {
    if (n < 0 && a.err) *a.err = 1;
    return false;
  }
  if (c0 < 0 || c1 > a.tokens || n > len) {
    if (a.err) *a.err = 1;
    return false;
  }
  const int64_t start = len - n;
  const int64_t page = (start >> lg) + j;
  if (page > (len - 1) >> lg) return false;
  if (page >= a.table_width) {
    if (a.err) *a.err = 1;
    return false;
  }
  const int64_t lo = start > (page << lg) ? start : page << lg;
  const int64_t hi = len < ((page + 1) << lg) ? len : (page + 1) << lg;
  g.row0 = c0 + (lo - start);
  g.index0 = lo;
  g.entry = a.table + (int64_t)b * a.table_stride + page;
  g.slot0 = (int)(lo - (page << lg));
  g.n = (int)(hi - lo);
  return true;
}

// Item i of the list of (sequence, touched page): sequence b's span begins at cu[b] / page + 2 b and is never
// shorter than the pages it touches, (n_b - 2) / page + 2 at most, so the list needs no prefix sum.
__device__ __forceinline__ bool find_segment(const AppendArgs& a, int64_t item, Segment& g) {
  const int lg = a.page_log2;
  const int b = find_sequence(a.seqs, item, [&](int i) { return ((int64_t)a.cu[i] >> lg) + 2 * (int64_t)i; });
  const int64_t c0 = a.cu[b];
  return segment_of(a, b, c0, item - ((c0 >> lg) + 2 * (int64_t)b), g);
}

// The segment's page, -1 where it does not exist.  (Looked up after the rows' loads have been issued.)
__device__ __forceinline__ int64_t page_of(const AppendArgs& a, const Segment& g) {
  const int64_t id = *g.entry;
  if (id >= 0 && id < a.num_pages) return id;
  if (a.err) *a.err = 1;
  return -1;
}

// A lane's 16 elements of a row as they are stored, and as fp32.
template <int DT>
struct Row {
  u32x4_t w[DT == PDM_F32 ? 4 : 2];
};

template <int DT, bool VEC>
__device__ __forceinline__ void load_row(const AppendArgs& a, int kv, int h, int64_t row, const RowPlace& pl, Row<DT>& x) {
  const int64_t at = row * a.stride_t[kv] + h * a.stride_h[kv];
  load8_raw<DT, VEC>(a.x[kv], at + pl.lo, x.w);
  load8_raw<DT, VEC>(a.x[kv], at + pl.hi, x.w + (DT == PDM_F32 ? 2 : 1));
}

template <int DT>
__device__ __forceinline__ void to_float(const Row<DT>& x, float* v) {
  raw_to_float<DT>(x.w, v);
  raw_to_float<DT>(x.w + (DT == PDM_F32 ? 2 : 1), v + 8);
}

// x in fp32, rounded to odd: what is cut off leaves the last bit set, so that the code's rounding sees on which side of a tie
// x lies.  (On the words of the double: 4 integer operations, where a comparison with the rounded number cost 1 us of 15.)
__device__ __forceinline__ float to_odd(double x) {
  constexpr uint32_t cut = 0x1fffffffu;  // the 29 bits that fp32 does not have
  const uint64_t bits = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = (uint32_t)bits;
  const uint64_t odd = (bits >> 32) << 32 | ((lo | ((lo & cut) + cut)) & ~cut);
  return (float)__builtin_bit_cast(double, odd);
}

// A key row normed and rotated, in 64 bits: its code is the nearest to the key itself, whatever the order of the sum.
// (Against 32 bits, in a kernel that took keys and values in two passes, the prompts above went from 35 to 49 us.)  Called by
// the row's whole group; `ok`: this row exists.
template <bool NORM, bool INTER>
__device__ __forceinline__ void key_row(const AppendArgs& a, const Segment& g, int r, bool ok, int j, const RowPlace& pl, float* v) {
  double rs = 1.0;
  if (NORM) {
    double ss = 0.0;
    if (ok) {
#pragma unroll
      for (int e = 0; e < 16; ++e) ss = __builtin_fma((double)v[e], (double)v[e], ss);
    }
    for (int o = 1; o < 1 << a.width_log2; o <<= 1) ss += __shfl_xor(ss, o);
    rs = 1.0 / sqrt(ss / (double)a.D + (double)a.eps);
  }
  if (!ok) return;
  float w[16], c[8], s[8];
  if (NORM) {
    load8f(a.w + pl.lo, w);
    load8f(a.w + pl.hi, w + 8);
  }
  bool zero = false;
  if (a.R > 0) {  // (also behind the rotated part: outside the tables the whole key is zero)
    const int64_t p = a.positions ? load_position(a.positions, a.bits, g.row0 + r) : g.index0 + r;
    zero = p < 0 || p >= a.table_rows;
    if (zero) {
      if (a.err) *a.err = 1;
    } else if (pl.turned) {
      load8f(a.cos + p * (a.R / 2) + 8 * j, c);
      load8f(a.sin + p * (a.R / 2) + 8 * j, s);
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int ia = INTER ? 2 * i : i, ib = INTER ? 2 * i + 1 : i + 8;
    double x = v[ia], y = v[ib];
    if (NORM) x = x * rs * (double)w[ia], y = y * rs * (double)w[ib];
    if (pl.turned) {
      const double t = x * (double)c[i] - y * (double)s[i];
      y = y * (double)c[i] + x * (double)s[i];
      x = t;
    }
    v[ia] = zero ? 0.0f : to_odd(x);
    v[ib] = zero ? 0.0f : to_odd(y);
  }
}

// Largest finite magnitude.  (fmaxf passes over NaN; an infinity is rare.)
__device__ __forceinline__ float row_max(const float* v) {
  float m = 0.0f;
#pragma unroll
  for (int e = 0; e < 16; ++e) m = fmaxf(m, fabsf(v[e]));
  if (m == __builtin_inff()) {
    m = 0.0f;
#pragma unroll
    for (int e = 0; e < 16; ++e) m = fmaxf(m, fabsf(v[e]) < __builtin_inff() ? fabsf(v[e]) : 0.0f);
  }
  return m;
}

// The exponent of a page's head for new values of at most `amax`, its own if that is larger (`slot0` tokens are there already
// and `held` is their exponent); codes that are there are brought to a larger one, thread `tid` of `threads`.
__device__ __forceinline__ int settle_scale(float amax, int slot0, int held, uint8_t* page, int D, int tid, int threads) {
  const int e = scale_exponent(amax);
  if (slot0 == 0) return e;
  if (e <= held) return held;
  const float f = exp2_int(held - e > -126 ? held - e : -126);
  for (int i = tid; i < slot0 * D / 16; i += threads) {
    u32x4_t* p = reinterpret_cast<u32x4_t*>(page) + i;
    u32x4_t c = *p;
#pragma unroll
    for (int d = 0; d < 4; ++d) {
      const f32x2_t lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[d], false);
      const f32x2_t hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[d], true);
      const float x[4] = {lo[0] * f, lo[1] * f, hi[0] * f, hi[1] * f};
      c[d] = e4m3x4(x);
    }
    *p = c;
  }
  return e;
}

__device__ __forceinline__ void store_codes(uint8_t* row, const RowPlace& pl, float* v, int e) {
  const float inv = exp2_int(-e);
#pragma unroll
  for (int d = 0; d < 16; ++d) v[d] *= inv;
  if (e == kScaleExpMax) {
#pragma unroll
    for (int d = 0; d < 16; ++d) v[d] = e4m3_saturated(v[d]);
  }
  *reinterpret_cast<u32x2_t*>(row + pl.lo) = u32x2_t{e4m3x4(v), e4m3x4(v + 4)};
  *reinterpret_cast<u32x2_t*>(row + pl.hi) = u32x2_t{e4m3x4(v + 8), e4m3x4(v + 12)};
}

// Pages with several new tokens: a page and head, its keys and then its values, per W waves; a lane group takes NI rows.  The
// loads of both are in flight together, and the values stay in registers between the maximum and the codes.
template <int DT, bool NORM, bool INTER, bool VEC, int W, int NI>
__device__ __forceinline__ void append_page(const AppendArgs& a, const Segment& g, int h) {
  __shared__ float red[2][4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int width = 1 << a.width_log2;
  const int j = lane & (width - 1);
  const int per_wave = 64 >> a.width_log2;
  const int group = (W == 4 ? wave * per_wave : 0) + (lane >> a.width_log2), groups = W * per_wave;
  const RowPlace pk = row_place<INTER>(j, a.D, a.R), pv = row_place<false>(j, a.D, a.D);
  Row<DT> xk[NI], xv[NI];
#pragma unroll
  for (int i = 0; i < NI; ++i)
    if (group + i * groups < g.n) load_row<DT, VEC>(a, 0, h, g.row0 + group + i * groups, pk, xk[i]);
#pragma unroll
  for (int i = 0; i < NI; ++i)
    if (group + i * groups < g.n) load_row<DT, VEC>(a, 1, h, g.row0 + group + i * groups, pv, xv[i]);
  const int64_t id = page_of(a, g);
  if (id < 0) return;
  const int64_t entry = id * a.heads + h;
  int held[2] = {0, 0};
  if (g.slot0 > 0) held[0] = scale_exponent_of(a.scale[0][entry]), held[1] = scale_exponent_of(a.scale[1][entry]);
  // the exponent of keys (0) or values (1)
  auto settle = [&](int kv, float amax) {
    amax = group_max(amax, 64);
    if (W == 4) {  // (and every wave has read the old scale)
      if (lane == 0) red[kv][wave] = amax;
      __syncthreads();
      amax = fmaxf(fmaxf(red[kv][0], red[kv][1]), fmaxf(red[kv][2], red[kv][3]));
    }
    const int e = settle_scale(amax, g.slot0, held[kv], a.codes[kv] + ((entry << a.page_log2) * a.D), a.D,
                               W == 4 ? threadIdx.x : lane, 64 * W);
    if (lane == 0 && (W == 1 || wave == 0)) a.scale[kv][entry] = exp2_int(e);
    return e;
  };
  const int64_t slots = (entry << a.page_log2) + g.slot0;
  {
    float v[NI][16], amax = 0.0f;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int r = group + i * groups;
      to_float(xk[i], v[i]);
      if (NORM || a.R > 0) key_row<NORM, INTER>(a, g, r, r < g.n, j, pk, v[i]);
      if (r < g.n) amax = fmaxf(amax, row_max(v[i]));
    }
    const int e = settle(0, amax);
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int r = group + i * groups;
      if (r < g.n) store_codes(a.codes[0] + (slots + r) * a.D, pk, v[i], e);
    }
  }
  float amax = 0.0f;
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    float v[16];
    to_float(xv[i], v);
    if (group + i * groups < g.n) amax = fmaxf(amax, row_max(v));
  }
  const int e = settle(1, amax);
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int r = group + i * groups;
    float v[16];
    to_float(xv[i], v);
    if (r < g.n) store_codes(a.codes[1] + (slots + r) * a.D, pv, v, e);
  }
}

// Sets the flag for spans of 256 sequences that do not fit.  The list above need not lead to them: a first span may lie behind
// the batch, one that runs backwards may be passed over.
__device__ __forceinline__ void check_spans(const AppendArgs& a, int64_t first) {
  const int64_t b = first + threadIdx.x;
  if (!a.err || b >= a.seqs) return;
  const int64_t c0 = a.cu[b], c1 = a.cu[b + 1];
  if (c1 != c0 && (c0 < 0 || c1 < c0 || c1 > a.tokens || c1 - c0 > a.lens[b])) *a.err = 1;
}

// (behind the first `blocks` workgroups those that check the spans)
template <int DT, bool NORM, bool INTER, bool VEC, int W, int NI>
__global__ void __launch_bounds__(256) kv_append_kernel(AppendArgs a, int64_t items, int64_t blocks) {
  const int64_t block = linear_block();
  if (block >= blocks) return check_spans(a, (block - blocks) * 256);
  const int64_t unit = (block * 4 + (threadIdx.x >> 6)) / W;
  const int64_t item = unit / a.heads;
  if (item >= items) return;  // W == 4: the same for the whole block
  Segment g;
  if (find_segment(a, item, g)) append_page<DT, NORM, INTER, VEC, W, NI>(a, g, (int)(unit - item * a.heads));
}

// Pages with a token or two: a lane group per (page, head, keys or values), its rows one after the other, read again for the
// codes where there are two.
constexpr int kFewTokens = 2;

template <int DT, bool NORM, bool INTER, bool VEC>
__device__ __forceinline__ void append_tokens(const AppendArgs& a, int64_t items, int waves, int64_t block) {
  const int lane = threadIdx.x & 63;
  const int64_t unit = block * 4 + (threadIdx.x >> 6);
  const int64_t item = unit / waves;
  if (item >= items) return;
  Segment g;
  if (!find_segment(a, item, g) || g.n > kFewTokens) return;
  const int width = 1 << a.width_log2, j = lane & (width - 1);
  const int part = (int)(unit - item * waves) * (64 >> a.width_log2) + (lane >> a.width_log2);
  const bool live = part < 2 * a.heads;
  const int kv = live && part >= a.heads, h = !live ? 0 : kv ? part - a.heads : part;
  const RowPlace pl = row_place<INTER>(j, a.D, a.R);  // (the values' pieces may be the keys')
  float x[16], amax = 0.0f;
  auto row = [&](int r) {
    if (!live) return;
    Row<DT> w;
    load_row<DT, VEC>(a, kv, h, g.row0 + r, pl, w);
    to_float(w, x);
  };
  auto key = [&](int r) {
    if (NORM || a.R > 0) {
      if (live && !kv) key_row<NORM, INTER>(a, g, r, true, j, pl, x);
    }
  };
  row(0);
  const int64_t id = page_of(a, g);
  if (id < 0) return;
  const int64_t entry = id * a.heads + h;
  const int held = g.slot0 > 0 && live ? scale_exponent_of(a.scale[kv][entry]) : 0;
  key(0);
  if (live) amax = row_max(x);
  for (int r = 1; r < g.n; ++r) {
    row(r);
    key(r);
    if (live) amax = fmaxf(amax, row_max(x));
  }
  amax = group_max(amax, width);
  if (!live) return;
  uint8_t* page = a.codes[kv] + ((entry << a.page_log2) * a.D);
  const int e = settle_scale(amax, g.slot0, held, page, a.D, j, width);
  if (j == 0) a.scale[kv][entry] = exp2_int(e);
  for (int r = g.n - 1; r >= 0; --r) {  // the last row is still there
    if (r < g.n - 1) {
      row(r);
      key(r);
    }
    store_codes(page + (int64_t)(g.slot0 + r) * a.D, pl, x, e);
  }
}

// The pages with more tokens of 256 sequences, by kParts workgroups: they look at the sequences, not at each page and head, so
// that a batch without any pays little (single tokens of 4,096 sequences 28 us; 95 with a workgroup for every page and head).
// The pages and heads of all busy sequences are dealt to them in turn: 3 tokens of each of 85 sequences, nothing of 171, 51 us
// (382 where each sequence's pages began with the first workgroup, 99 with 64 of them), 6 heads of 64 12 us (360, 17).
constexpr int kParts = 128;

template <int DT, bool NORM, bool INTER, bool VEC, int W, int NI>
__device__ __forceinline__ void append_busy(const AppendArgs& a, int64_t block) {
  __shared__ int before[256], sums[4];  // pages before a sequence's, and of a wave's sequences
  const int64_t first = block / kParts * 256;
  const int part = (int)(block % kParts), lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t mine = first + threadIdx.x;
  if (part == 0) check_spans(a, first);
  int pages = 0;  // that the sequence's tokens may touch
  if (mine < a.seqs) {
    const int64_t c0 = a.cu[mine], c1 = a.cu[mine + 1], n = c1 - c0;
    if (n > kFewTokens && c0 >= 0 && c1 <= a.tokens && n <= a.lens[mine]) pages = (int)(n - 2 >> a.page_log2) + 2;
  }
  if (!__syncthreads_or(pages)) return;
  int upto = pages;
  for (int o = 1; o < 64; o <<= 1) {
    const int v = __shfl_up(upto, o);
    upto += lane >= o ? v : 0;
  }
  if (lane == 63) sums[wave] = upto;
  __syncthreads();
  int all = 0;
  for (int w = 0; w < 4; ++w) {
    if (w < wave) upto += sums[w];
    all += sums[w];
  }
  before[threadIdx.x] = upto - pages;
  __syncthreads();
  // (W == 4: the same for the whole block, and what a turn leaves in LDS is read before the next one's first barrier)
  for (int64_t u = part * (4 / W) + (W == 4 ? 0 : wave); u < (int64_t)all * a.heads; u += kParts * (4 / W)) {
    const int page = (int)(u / a.heads), i = find_sequence(256, page, [&](int x) { return before[x]; });
    const int b = (int)first + i;
    Segment g;
    if (segment_of(a, b, a.cu[b], page - before[i], g) && g.n > kFewTokens)
      append_page<DT, NORM, INTER, VEC, W, NI>(a, g, (int)(u - (int64_t)page * a.heads));
  }
}

// A batch of single tokens, as a rule; a sequence with more has its pages in the workgroups behind the first `few`.
template <int DT, bool NORM, bool INTER, bool VEC, int W, int NI>
__global__ void __launch_bounds__(256) kv_append_token_kernel(AppendArgs a, int64_t items, int waves, int64_t few, int64_t all) {
  const int64_t block = linear_block();
  if (block < few) append_tokens<DT, NORM, INTER, VEC>(a, items, waves, block);
  else if (block < all) append_busy<DT, NORM, INTER, VEC, W, NI>(a, block - few);
}

template <int DT, bool NORM, bool INTER, bool VEC, int W, int NI>
void launch_kernel(const AppendArgs& a, int64_t items, hipStream_t st) {
  // 64 sequences behind 100 tokens each, 8 heads of 128, pages of 64: one token each 5.7 us in the first kernel, 8.0 in the
  // second; two each 8.2 and 7.7; 64 tokens of one sequence 8.9 (151 where lane groups take them row by row); single tokens of
  // 4,096 sequences 28
  if (a.tokens <= a.seqs) {
    const int parts = 64 >> a.width_log2, waves = (2 * a.heads + parts - 1) / parts;
    const int64_t few = (items * waves + 3) / 4, all = few + ((int64_t)a.seqs + 255) / 256 * kParts;
    kv_append_token_kernel<DT, NORM, INTER, VEC, W, NI><<<linear_grid(all), 256, 0, st>>>(a, items, waves, few, all);
  } else {
    const int64_t blocks = (items * a.heads * W + 3) / 4, all = blocks + ((int64_t)a.seqs + 255) / 256;
    kv_append_kernel<DT, NORM, INTER, VEC, W, NI><<<linear_grid(all), 256, 0, st>>>(a, items, blocks);
  }
}

template <int DT, bool NORM, bool INTER, bool VEC>
int launch(const AppendArgs& a, hipStream_t st) {
  const int64_t items = (a.tokens >> a.page_log2) + 2 * (int64_t)a.seqs;
  // rows of a page per wave-wide step; more than 4 of them take the four waves of a block
  const int steps = (1 << a.page_log2) * (1 << a.width_log2) / 64;
  if (steps <= 1) launch_kernel<DT, NORM, INTER, VEC, 1, 1>(a, items, st);
  else if (steps == 2) launch_kernel<DT, NORM, INTER, VEC, 1, 2>(a, items, st);
  else if (steps == 4) launch_kernel<DT, NORM, INTER, VEC, 4, 1>(a, items, st);
  else if (steps == 8) launch_kernel<DT, NORM, INTER, VEC, 4, 2>(a, items, st);
  else if (steps == 16) launch_kernel<DT, NORM, INTER, VEC, 4, 4>(a, items, st);
  else launch_kernel<DT, NORM, INTER, VEC, 4, 8>(a, items, st);
  PDM_CHECK_LAUNCH();
  return PDM_OK;
}

template <int DT, bool NORM>
int launch2(bool inter, bool vec, const AppendArgs& a, hipStream_t st) {
  if (inter) return vec ? launch<DT, NORM, true, true>(a, st) : launch<DT, NORM, true, false>(a, st);
  return vec ? launch<DT, NORM, false, true>(a, st) : launch<DT, NORM, false, false>(a, st);
}

template <int DT>
int launch1(bool norm, bool inter, bool vec, const AppendArgs& a, hipStream_t st) {
  return norm ? launch2<DT, true>(inter, vec, a, st) : launch2<DT, false>(inter, vec, a, st);
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace
}  // namespace pdm

using namespace pdm;

extern "C" int pdm_kv_append(const pdm_kv_append_desc* d, const pdm_kv_cache* cache, const pdm_kv_batch* batch,
                             const void* k, const void* v, const void* positions, const float* cos, const float* sin,
                             const float* k_weight, int32_t* err_flag, pdm_stream_t stream) {
  clear_error();
  PDM_CHECK_ARG(d && cache && batch, "null descriptor");
  if (int e = check_cache(__func__, cache, batch)) return e;
  PDM_CHECK_ARG(d->dtype == PDM_F32 || d->dtype == PDM_F16 || d->dtype == PDM_BF16, "dtype must be F32, F16 or BF16");
  PDM_CHECK_ARG(d->rotary_dim >= 0 && d->rotary_dim <= cache->head_dim && d->rotary_dim % 16 == 0,
                "rotary_dim must be a multiple of 16 in [0, head_dim]");
  PDM_CHECK_ARG(d->position_bits == 32 || d->position_bits == 64, "position_bits must be 32 or 64");
  PDM_CHECK_ARG(d->table_rows >= 0 && d->eps >= 0, "negative table_rows or eps");
  if (batch->tokens == 0 || batch->num_seqs == 0) return PDM_OK;
  PDM_CHECK_ARG(k && v, "null k / v");
  PDM_CHECK_ARG(!d->rotary_dim || (cos && sin), "null cos / sin");
  PDM_CHECK_ARG(aligned16(cos) && aligned16(sin) && aligned16(k_weight), "cos, sin and weight must be 16-byte aligned");
  const int64_t unit = d->dtype == PDM_F32 ? 4 : 8;
  const bool vec = aligned16(k) && aligned16(v) && d->k_stride_t % unit == 0 && d->k_stride_h % unit == 0 &&
                   d->v_stride_t % unit == 0 && d->v_stride_h % unit == 0;
  AppendArgs a{};
  a.x[0] = k, a.x[1] = v;
  a.stride_t[0] = d->k_stride_t, a.stride_t[1] = d->v_stride_t;
  a.stride_h[0] = d->k_stride_h, a.stride_h[1] = d->v_stride_h;
  a.codes[0] = cache->k_codes, a.codes[1] = cache->v_codes;
  a.scale[0] = cache->k_scale, a.scale[1] = cache->v_scale;
  a.cu = batch->cu_seqlens, a.table = batch->page_table, a.lens = batch->seq_lens;
  a.positions = positions;
  a.cos = cos, a.sin = sin, a.w = k_weight, a.err = err_flag;
  a.tokens = batch->tokens, a.table_stride = batch->table_stride, a.table_rows = d->table_rows;
  a.num_pages = cache->num_pages;
  a.seqs = batch->num_seqs, a.heads = cache->n_kv_heads, a.D = cache->head_dim, a.R = d->rotary_dim;
  a.page_log2 = log2_of(cache->page_size), a.table_width = batch->table_width, a.bits = d->position_bits;
  a.width_log2 = log2_of(cache->head_dim / 16);
  a.eps = d->eps;
  const bool norm = k_weight != nullptr, inter = d->interleaved != 0;
  if (d->dtype == PDM_F32) return launch1<PDM_F32>(norm, inter, vec, a, stream);
  if (d->dtype == PDM_F16) return launch1<PDM_F16>(norm, inter, vec, a, stream);
  return launch1<PDM_BF16>(norm, inter, vec, a, stream);
}
