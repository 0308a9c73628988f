// Device helpers of the attention of ragged batches (jagged_attention.hip, jagged_backward.hip): sequences and the keys
// that their queries see, tiles in LDS and their fragments, the bias by distance.
#pragma once

#include "kv_common.h"

namespace pdm {

typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
typedef short s16x4_t __attribute__((ext_vector_type(4)));

struct JagArgs {
  const void *q, *k, *v;
  const int32_t *cu_q, *cu_k;
  const float* bias;                 // [hq, bias_last + 1] or null
  int32_t* err;
  void *out, *rest;                  // forward; rest: what rounding out left, see rest2 (may be null)
  float *lse, *stats;                // stats: a row's reference (log2) and 1 / the sum of its weights
  float* outer;                      // a row's weights of the bias's last column and of what lies before its first, or null
  const void* dout;                  // backward
  const float* dlse;
  void *dq, *dk, *dv;
  float* dbias;
  float* delta;                      // sum_d dout out - dlse, [q_tokens, hq]
  int32_t* expo;                     // fp16: exponent of the largest |dout| of 32 rows, [items of 128 rows, 4, hq]
  float* part;                       // partial gradients of the bias, [items of 128 rows, hq, part_stride]
  int32_t* part_range;               // [items, 2]: the distances that a partial gradient holds
  float* sink_part;                  // sums of the gradients of sinks, see jag_dkv_kernel
  int32_t sink_cell, sink_rows, sink_list, sink_blocks, sink_shares;
  int64_t part_stride;
  int64_t q_tokens, k_tokens, items;
  int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh;
  int32_t seqs, hq, hk, group, causal, window, sinks, bias_start, bias_last;
  float scale, scale2;               // scale2 = scale * log2(e)
};

constexpr float kInf = __builtin_inff();
constexpr float kNoKeys = 3e38f;  // the reference of a row without weights: none passes it
constexpr float kLargeScore = 0x1p12f;
constexpr float kLn2 = 0.69314718055994531f, kLog2e = 1.44269504088896341f;

// A kernel's arguments, read again: those that its end alone needs else take scalar registers all the way, and others are held in
// lanes for them.  (JagArgs is every kernel's first argument.)
__device__ __forceinline__ const JagArgs& late_args() {
  typedef const __attribute__((address_space(4))) JagArgs* Constant;
  Constant p = (Constant)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return *(const JagArgs*)p;
}

// ---- sequences -------------------------------------------------------------------
struct JagSeq {
  int64_t q0, k0;  // its first rows
  int nq, nk;
};

// False where the spans do not fit the batch.
__device__ __forceinline__ bool jag_seq(const JagArgs& a, int b, JagSeq& s) {
  const int64_t c0 = a.cu_q[b], c1 = a.cu_q[b + 1], k0 = a.cu_k[b], k1 = a.cu_k[b + 1];
  s.q0 = c0, s.k0 = k0, s.nq = (int)(c1 - c0), s.nk = (int)(k1 - k0);
  return c0 >= 0 && c0 <= c1 && c1 <= a.q_tokens && k0 >= 0 && k0 <= k1 && k1 <= a.k_tokens;
}

// Block `item` of the list of (sequence, M rows of the spans `cu`): sequence b's part of it begins at cu[b] / M + b.
// False for an item without rows.
template <int M>
__device__ __forceinline__ bool jag_block(const JagArgs& a, const int32_t* cu, int64_t item, JagSeq& s, int& b, int& r0) {
  b = find_sequence(a.seqs, item, [&](int i) { return (int64_t)cu[i] / M + i; });
  const int64_t j = item - ((int64_t)cu[b] / M + b);
  if (j < 0 || !jag_seq(a, b, s) || j * M >= (cu == a.cu_q ? s.nq : s.nk)) return false;
  r0 = (int)(j * M);
  return true;
}

// Sum over the wave, for all of it: shifts within rows of 16 lanes, then rows on rows.
__device__ __forceinline__ int wave_sum(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, true);  // from 1, 2, 4 and 8 lanes below
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // the last lane of a row to the next
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // lane 31 to the upper rows
  return __builtin_amdgcn_readlane(x, 63);
}

// The same list with the blocks that take longest first, for batches of at most 64 sequences, whose workgroups are few beside the
// places for them: a late long one would be waited for (training on 8 sequences of 1,001 to 2,777 tokens: 633 -> 557 us).  A
// block's cost goes by its level: causal, its number in the sequence, from the other end for blocks of keys (`keys`); else its
// sequence's length.  Every lane has a sequence; the level of a rank is found by halving over sums of the wave.
template <int M>
__device__ __forceinline__ bool jag_ranked_block(const JagArgs& a, bool keys, int64_t rank, JagSeq& s, int& b, int& r0) {
  const int lane = threadIdx.x & 63;
  JagSeq mine{};
  int n = 0;  // blocks of this lane's sequence
  if (lane < a.seqs && jag_seq(a, lane, mine)) n = ((keys ? mine.nk : mine.nq) + M - 1) / M;
  auto above = [&](int level) { return wave_sum(a.causal ? (n - 1 > level ? n - 1 - level : 0) : (n - 1 > level ? n : 0)); };  // blocks of higher levels
  if (rank >= above(-1)) return false;
  int lo = 0, hi = 1;  // the level: the lowest with above(level) <= rank
  while (__ballot(n > hi)) hi *= 2;
  --hi;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (above(mid) <= rank) hi = mid;
    else lo = mid + 1;
  }
  const int at = (int)rank - above(lo), each = a.causal ? 1 : lo + 1;  // place in the level; blocks that a sequence has there
  const unsigned long long in = __ballot(a.causal ? n > lo : n == lo + 1);
  const int before = __builtin_popcountll(in & ((1ull << lane) - 1));
  b = __builtin_ctzll(__ballot((in >> lane & 1) && before == at / each));
  const int blocks = __builtin_amdgcn_readlane(n, b);
  r0 = (a.causal ? (keys ? blocks - 1 - lo : lo) : at % each) * M;
  s.q0 = __builtin_amdgcn_readlane((int)mine.q0, b), s.k0 = __builtin_amdgcn_readlane((int)mine.k0, b);
  s.nq = __builtin_amdgcn_readlane(mine.nq, b), s.nk = __builtin_amdgcn_readlane(mine.nk, b);
  return true;
}

// Rows [first, first + 256) of the batch that no sequence which fits covers are given to clear(row), one after the other, by
// the whole block of 256 threads; sequences [first, first + 256) that do not fit set the flag.
template <typename F>
__device__ __forceinline__ void jag_guard(const JagArgs& a, const int32_t* cu, int64_t tokens, int64_t first, F clear) {
  __shared__ uint8_t bad[256];
  const int64_t t = first + threadIdx.x;
  JagSeq s;
  if (t < a.seqs && !jag_seq(a, (int)t, s) && a.err) *a.err = 1;
  bool covered = false;
  if (t < tokens && a.seqs > 0) {
    int lo = 0, hi = a.seqs;  // last b with cu[b] <= t
    while (hi - lo > 1) {
      const int mid = lo + (hi - lo) / 2;
      if (cu[mid] <= t) lo = mid;
      else hi = mid;
    }
    covered = cu[lo] <= t && t < cu[lo + 1] && jag_seq(a, lo, s);
  }
  const bool open = t < tokens && !covered;
  bad[threadIdx.x] = open;
  if (!__syncthreads_or(open)) return;
  for (int r = 0; r < 256 && first + r < tokens; ++r)
    if (bad[r]) clear(first + r);
}

__device__ __forceinline__ void clear_row(void* base, int64_t at, int elements) {  // of 16 bits; 16-byte aligned, all of a block
  u32x4_t* p = reinterpret_cast<u32x4_t*>(static_cast<uint16_t*>(base) + at);
  for (int i = threadIdx.x; i < elements / 8; i += 256) p[i] = u32x4_t{0, 0, 0, 0};
}

// ---- what a block of queries sees ------------------------------------------------------
// Tiles of KT keys: those of the first tokens that stay visible, then [lo, hi), lo a multiple of KT.
struct JagKeys {
  int lo, hi, first, tiles;  // first: tiles before lo
};
template <int KT>
__device__ __forceinline__ JagKeys jag_keys(const JagArgs& a, const JagSeq& s, int i0, int i1) {  // queries i0 .. i1
  const int p0 = s.nk - s.nq + i0, p1 = s.nk - s.nq + i1;
  JagKeys k;
  k.hi = a.causal && p1 + 1 < s.nk ? p1 + 1 : s.nk;
  if (k.hi < 0) k.hi = 0;
  k.lo = a.window > 0 && p0 - a.window + 1 > 0 ? (p0 - a.window + 1) & ~(KT - 1) : 0;
  if (k.lo > k.hi) k.lo = (k.hi + KT - 1) & ~(KT - 1);
  const int sinks = a.sinks < k.hi ? a.sinks : k.hi;
  k.first = (sinks + KT - 1) / KT;
  if (k.first * KT >= k.lo) k.first = 0, k.lo = sinks > 0 ? 0 : k.lo;
  k.tiles = k.first + (k.hi > k.lo ? (k.hi - k.lo + KT - 1) / KT : 0);
  return k;
}
template <int KT>
__device__ __forceinline__ int jag_key(const JagKeys& k, int t) { return t < k.first ? t * KT : k.lo + (t - k.first) * KT; }

// ---- types -----------------------------------------------------------------------------
template <int DT>
__device__ __forceinline__ f32x16_t mfma32(u32x4_t a, u32x4_t b, f32x16_t c) {
  if constexpr (DT == PDM_BF16) return mfma32x32x16(a, b, c);
  else return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
}
template <int DT>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {  // nearest even
  if constexpr (DT == PDM_BF16) return pack_bf16x2(lo, hi);
  else return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2_t{lo, hi}, f16x2_t));
}
template <int DT>
__device__ __forceinline__ float lo_of(uint32_t w) {
  return DT == PDM_BF16 ? __uint_as_float(w << 16) : f16_bits_to_f32(w & 0xffffu);
}
template <int DT>
__device__ __forceinline__ float hi_of(uint32_t w) {
  return DT == PDM_BF16 ? __uint_as_float(w & 0xffff0000u) : f16_bits_to_f32(w >> 16);
}
template <int DT>
__device__ __forceinline__ uint32_t left2(float lo, float hi, uint32_t w) {  // what rounding the pair to w left
  return pack2<DT>(lo - lo_of<DT>(w), hi - hi_of<DT>(w));
}
// What rounding a pair to w left, in 16 bits an element: fp16's remainders; of bf16 the lower halves of the fp32 bits, which lose
// nothing (a remainder in bf16 leaves 2^-18, which would be most of the error of the bias's gradient).  Of halves of 0x8000 w does not
// tell which way they were rounded: these are moved by one.
template <int DT>
__device__ __forceinline__ uint32_t rest2(float lo, float hi, uint32_t w) {
  if constexpr (DT == PDM_F16) return left2<DT>(lo, hi, w);
  auto half = [](uint32_t bits) {
    const uint32_t x = bits & 0xffffu;
    return x == 0x8000u ? 0x7fffu + 2 * (bits >> 16 & 1) : x;
  };
  return half(__float_as_uint(lo)) | half(__float_as_uint(hi)) << 16;
}
// The remainder of the lower (upper) element of w.
template <int DT>
__device__ __forceinline__ float rest_lo(uint32_t w, uint32_t rest) {
  if constexpr (DT == PDM_F16) return lo_of<DT>(rest);
  const uint32_t r = rest & 0xffffu;
  return __uint_as_float(((w << 16) - ((r >> 15) << 16)) | r) - lo_of<DT>(w);
}
template <int DT>
__device__ __forceinline__ float rest_hi(uint32_t w, uint32_t rest) { return rest_lo<DT>(w >> 16, rest >> 16); }
// Bits 15 and 31: the element there is infinite or NaN.
template <int DT>
__device__ __forceinline__ uint32_t odd2(uint32_t w) {
  constexpr uint32_t E = DT == PDM_BF16 ? 0x7f807f80u : 0x7c007c00u, U = DT == PDM_BF16 ? 0x00800080u : 0x04000400u;
  return ((w & E) + U) & 0x80008000u;
}

// ---- tiles in LDS -----------------------------------------------------------------------
// Rows of D elements in pieces of 16 bytes; piece g of row r lies at place g ^ turn(r).  The rows of a fragment read then begin
// in different banks, and so do the 4 rows of 4 pieces that half a wave takes by a transposing read.
template <int D>
struct Tile {
  static constexpr int RS = 2 * D;
  __device__ static constexpr int turn(int r) {
    return D == 64 ? (r >> 1 & 1) << 2 | (r & 1) << 1 | (r >> 2 & 1) : (r & 3) << 2 | (r >> 2 & 3);
  }
  // A fragment's element i of lane l: row l % 32, column 16 kk + 8 (l / 32) + i.
  static __device__ __forceinline__ uint32_t row_at(int lane) { return (lane & 31) * RS + 16 * (lane >> 5 ^ turn(lane & 31)); }
  static __device__ __forceinline__ u32x4_t rows(const char* t, uint32_t at, int row, int kk) {
    return *reinterpret_cast<const u32x4_t*>(t + (at ^ (32 * kk)) + row * RS);
  }
  // Transposed: lane l has column 32 d + l % 32 of the 8 rows y + 4 (l / 32) + {0 .. 3, 8 .. 11}, which is the order in
  // which a 32x32 product leaves its rows.  A read of 16 lanes transposes 4 rows of 16 elements.
  static __device__ __forceinline__ uint32_t col_at(int lane) {
    const int r = 4 * (lane >> 5) + ((lane & 15) >> 2);
    return r * RS + 16 * ((2 * (lane >> 4 & 1) + (lane >> 1 & 1)) ^ turn(r)) + 8 * (lane & 1);
  }
  static __device__ __forceinline__ u32x4_t cols(const char* t, uint32_t at, int y, int d) {
    typedef __attribute__((address_space(3))) s16x4_t* lds_t;
    char* p = const_cast<char*>(t) + y * RS;
    const u32x2_t lo = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_t)(p + (at ^ (64 * d)))));
    const u32x2_t hi = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_t)(p + (at ^ (64 * d ^ 16 * turn(8))) + 8 * RS)));
    return u32x4_t{lo[0], lo[1], hi[0], hi[1]};
  }
};

// Eight elements, zeros where !there.
__device__ __forceinline__ u32x4_t load16(const uint16_t* p, bool there) {
  return there ? *reinterpret_cast<const u32x4_t*>(p) : u32x4_t{0, 0, 0, 0};
}

// A workgroup of 4 waves brings ROWS rows of a head into a tile without registers in between: buffer loads into LDS, whose lanes
// land 16 bytes apart, so that a lane takes the piece that belongs at its place.  Rows behind the n that are there come as zeros.
// Counted by vmcnt.
template <int D, int ROWS>
struct Bring {
  static constexpr int N = ROWS * D / 8 / 256;  // loads of a wave
  static constexpr int R = 64 / (D / 8);        // rows of a load
  uint32_t off[D == 64 ? 1 : N];                // of this lane's pieces, but for the rows of a load of D = 64
  uint32_t step;
  __device__ __forceinline__ void init(int64_t stride, int lane, int wave) {
    step = (uint32_t)stride * 2;
#pragma unroll
    for (int i = 0; i < (D == 64 ? 1 : N); ++i) {
      const int r = (wave * N + i) * R + lane / (D / 8);
      off[i] = r * step + 16 * ((lane % (D / 8)) ^ Tile<D>::turn(r));
    }
  }
  __device__ __forceinline__ void load(const uint16_t* head, int64_t stride, int row0, int n, const char* tile, int wave) const {
    const int rows = n - row0 < ROWS ? n - row0 : ROWS;
    const uint64_t base = reinterpret_cast<uint64_t>(head + row0 * stride);
    typedef uint32_t u32x4s __attribute__((ext_vector_type(4)));
    const u32x4s rsrc = {(uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)base), (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(base >> 32) & 0xffffu),
                         (uint32_t)__builtin_amdgcn_readfirstlane((rows - 1) * step + 2 * D), 0x00027000u};
    const uint32_t lds = __builtin_amdgcn_readfirstlane((uint32_t)reinterpret_cast<uintptr_t>(
        (__attribute__((address_space(3))) const char*)tile) + wave * N * 1024);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const uint32_t v = D == 64 ? off[0] + i * R * step : off[D == 64 ? 0 : i];
      asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds"
                   :: "v"(v), "s"(rsrc), "s"(lds + i * 1024) : "memory", "m0");
    }
  }
};
// This wave's loads into LDS have landed.
__device__ __forceinline__ void brought() { __builtin_amdgcn_s_waitcnt(kWaitVmcnt0); }

// A wave's own 32 rows of a head, [row0, row0 + 32) of n, into 32 rows of a tile.  (Fragments loaded from memory take 32 bytes of
// 32 lines an instruction, and lines fall out of the first cache between two of them.)
template <int D>
__device__ __forceinline__ void bring_own(const void* head, int64_t stride, int row0, int n, const char* tile) {
  constexpr int R = 64 / (D / 8);
  const int lane = threadIdx.x & 63, rows = n - row0 < 32 ? n - row0 : 32;
  const uint32_t step = (uint32_t)stride * 2;
  const uint64_t base = reinterpret_cast<uint64_t>(static_cast<const uint16_t*>(head) + row0 * stride);
  typedef uint32_t u32x4s __attribute__((ext_vector_type(4)));
  const u32x4s rsrc = {(uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)base), (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(base >> 32) & 0xffffu),
                       (uint32_t)__builtin_amdgcn_readfirstlane(rows > 0 ? (rows - 1) * step + 2 * D : 0), 0x00027000u};
  const uint32_t lds = __builtin_amdgcn_readfirstlane((uint32_t)reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) const char*)tile));
#pragma unroll
  for (int i = 0; i < 32 / R; ++i) {
    const int r = i * R + lane / (D / 8);
    const uint32_t v = r * step + 16 * ((lane % (D / 8)) ^ Tile<D>::turn(r));
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds"
                 :: "v"(v), "s"(rsrc), "s"(lds + i * 1024) : "memory", "m0");
  }
}

// What a wave writes to LDS and reads back itself: its LDS instructions take effect in order, the compiler must keep theirs.
__device__ __forceinline__ void own_lds_order() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local"); }

// ---- products with a tile's columns ------------------------------------------------------
// A weight of a pair that is not seen is zero, and what it meets must not matter, though 0 times an infinity or NaN would.  So
// where not every pair of a tile is seen, a wave looks at the rows that it brought, before the others read them, and puts zeros
// for such elements (clean_rows); behind the walk over all tiles, a second one over those tiles as they are brings them to the
// pairs that see them (mark_cols).

// True where rows that this wave brought held infinities or NaN; `rows`, where given, gets 1 for these (of ROWS) and 0 for its others.
template <int DT, int D, int ROWS>
__device__ __forceinline__ bool clean_rows(char* t, int lane, int wave, uint8_t* rows = nullptr) {
  constexpr int N = Bring<D, ROWS>::N, R = 64 / (D / 8);
  u32x4_t* p = reinterpret_cast<u32x4_t*>(t + wave * N * 1024 + lane * 16);
  uint32_t odd = 0;
  u32x4_t w[N];
#pragma unroll
  for (int i = 0; i < N; ++i) w[i] = p[64 * i];
#pragma unroll
  for (int i = 0; i < N; ++i) odd |= (odd2<DT>(w[i][0]) | odd2<DT>(w[i][1])) | (odd2<DT>(w[i][2]) | odd2<DT>(w[i][3]));
  if (!__any(odd != 0)) return false;
  if (rows && lane < N * R) rows[wave * N * R + lane] = 0;
#pragma unroll 1
  for (int i = 0; i < N; ++i) {
    u32x4_t x = p[64 * i];
    bool here = false;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t n = odd2<DT>(x[e]) >> 15;  // bits 0 and 16
      here = here || n != 0;
      x[e] &= ~((n << 16) - n);
    }
    p[64 * i] = x;
    if (rows && here) rows[(wave * N + i) * R + lane / (D / 8)] = 1;
  }
  return true;
}

// acc[d] += columns of rows [y0, y0 + 16 Y) of the tile, times w (the weights of these rows, as a 32x32 product left them);
// TWICE: and times rest.  Fragments are read LEAD products ahead.
template <int DT, int D, int Y, bool TWICE = false>
__device__ __forceinline__ void add_cols(f32x16_t* acc, const char* t, uint32_t at, int y0, const u32x4_t* w, const u32x4_t* rest = nullptr) {
  constexpr int N = Y * (D / 32), LEAD = 4;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int y = i / (D / 32), d = i % (D / 32);
    const u32x4_t f = Tile<D>::cols(t, at, y0 + 16 * y, d);
    acc[d] = mfma32<DT>(f, w[y], acc[d]);
    if constexpr (TWICE) acc[d] = mfma32<DT>(f, rest[y], acc[d]);
  }
  __builtin_amdgcn_sched_group_barrier(0x100, 2 * LEAD, 0);  // two LDS reads a fragment
#pragma unroll
  for (int i = 0; i < N - LEAD; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x008, TWICE ? 2 : 1, 0);
    __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
  }
  __builtin_amdgcn_sched_group_barrier(0x008, LEAD * (TWICE ? 2 : 1), 0);
}

// The second walk: products of 2^127 and 2, which no sum in fp32 holds, for pairs that are seen: +infinity, -infinity, and both for
// NaN, or for all of them (NANS: their weights are 0 or NaN).  sees(r): whether this lane's column sees row r of the tile.
template <int DT, int D, int Y, bool NANS, typename F>
__device__ __forceinline__ void mark_cols(f32x16_t* acc, const char* t, uint32_t at, int y0, F sees) {
  constexpr uint32_t pos = DT == PDM_BF16 ? 0x7f80u : 0x7c00u, neg = pos | 0x8000u;
  const int h4 = 4 * (threadIdx.x >> 5 & 1);
#pragma unroll 1
  for (int y = 0; y < Y; ++y) {
    u32x4_t seen;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int r = y0 + 16 * y + h4 + 8 * (e >> 1) + 2 * (e & 1);
      seen[e] = (sees(r) ? 0x4000u : 0u) | (sees(r + 1) ? 0x40000000u : 0u);  // bf16 2
    }
#pragma unroll
    for (int d = 0; d < D / 32; ++d) {
      const u32x4_t f = Tile<D>::cols(t, at, y0 + 16 * y, d);
      u32x4_t up, down;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t n = odd2<DT>(f[e]) >> 15, full = (n << 16) - n, x = f[e] & 0xffffu, z = f[e] >> 16;
        up[e] = full & ((!NANS && x == neg ? 0u : 0x7f00u) | (!NANS && z == neg ? 0u : 0x7f000000u));    // bf16 2^127
        down[e] = full & ((!NANS && x == pos ? 0u : 0xff00u) | (!NANS && z == pos ? 0u : 0xff000000u));
      }
      acc[d] = mfma32x32x16(up, seen, acc[d]);
      acc[d] = mfma32x32x16(down, seen, acc[d]);
    }
  }
}

// A wave's 32 columns of transposed sums, times f, to rows of 16-bit elements `stride` apart, of which n are there: through 32
// rows of a tile, so that whole lines are written.  LEFT: what the rounding left, to `left`.
template <int DT, int D, bool LEFT = false>
__device__ __forceinline__ void store_own(const f32x16_t* acc, float f, char* tile, void* base, void* left, int64_t at, int64_t stride, int n) {
  constexpr int R = 64 / (D / 8);
  const int lane = threadIdx.x & 63, c = lane & 31, h = lane >> 5;
#pragma unroll
  for (int pass = 0; pass < (LEFT ? 2 : 1); ++pass) {
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        float y[4];
        u32x2_t w;
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = acc[d][e + i] * f;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          w[i] = pack2<DT>(y[2 * i], y[2 * i + 1]);
          if (pass) w[i] = rest2<DT>(y[2 * i], y[2 * i + 1], w[i]);
        }
        *reinterpret_cast<u32x2_t*>(tile + c * Tile<D>::RS + 16 * ((4 * d + e / 4) ^ Tile<D>::turn(c)) + 8 * h) = w;
      }
    own_lds_order();
    uint16_t* to = static_cast<uint16_t*>(pass ? left : base) + at;
#pragma unroll
    for (int i = 0; i < 32 / R; ++i) {
      const int r = i * R + lane / (D / 8);
      const u32x4_t w = *reinterpret_cast<const u32x4_t*>(tile + i * 1024 + lane * 16);
      if (r < n) *reinterpret_cast<u32x4_t*>(to + r * stride + 8 * ((lane % (D / 8)) ^ Tile<D>::turn(r))) = w;
    }
    own_lds_order();
  }
}

// ---- the bias by distance -----------------------------------------------------------------
// Columns of a run of distances from d on, as a column that fits 32 bits with any key taken off: held where it makes no difference.
__device__ __forceinline__ int bias_from(const JagArgs& a, int64_t d) {
  const int64_t c = d - a.bias_start;
  return c < -(1 << 30) ? -(1 << 30) : c > 0x7fffff00 ? 0x7fffff00 : (int)c;
}
// Of column c (held within the bias) in units of log2, finite where the bias is.
__device__ __forceinline__ float bias2(const JagArgs& a, const float* row, int c) {
  const float b = row[(uint32_t)min(max(c, 0), a.bias_last)], v = b * kLog2e;
  return fabsf(b) < kInf ? __builtin_amdgcn_fmed3f(v, -3.402823466e38f, 3.402823466e38f) : v;
}

}  // namespace pdm
