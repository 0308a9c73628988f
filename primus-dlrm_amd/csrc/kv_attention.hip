// Attention of new tokens over an 8-bit paged cache.
//
// The rows of a (sequence, key head) are its new tokens times the query heads that share the key head, token by
// token; they meet the same keys, so a tile of 16 rows fills an MFMA whatever the mix of tokens and heads.
// Everything is transposed, S^T = K Q^T and O^T = V^T P^T: a lane then holds scores of one row (its column), the
// softmax needs no exchange between lanes but for a new maximum, and P^T is already in the layout of the second
// product's operand when the keys of a step are numbered as the first product leaves them.
//
// Codes become operands by conversion alone: e4m3 is a subset of bf16 and of f16, keys are converted bare and their
// page's scale is a factor of the scores in fp32, values are converted with their power-of-two scale, which bf16
// holds exactly.  f16 would not hold the values, so weights are bf16 as well, which leaves 2^-8 of a weight, half a step of a
// bf16 output and eight of an fp16 one.  So a weight goes in as a bf16 number and the bf16 remainder, 2^-16 of it left, by a
// second product with the same values: few rows, whose matrix units wait for the keys (63.4 -> 64.1 us for 64 sequences of 128
// to 8,192 tokens), and many rows of fp16 (794 -> 1,061 us for the prompts below).  Many rows of bf16 do without it: the error
// of their outputs goes from 1.7e-3, of the output's own rounding, to 2.1e-3, at 794 us instead of 1,048.  The running sum
// takes weights before any rounding.
//
// The simplest kernel, a wave for each (row, head), took 289 us for one sequence of 1,000 tokens, 4,764 for 64 of 128 to 8,192
// and 110,493 for two prompts of 4,000 tokens behind 4,000 (32 query heads, 8 key heads of 128); these take 9.6, 65 and 786.
#include <type_traits>

#include "kv_common.h"

namespace pdm {
namespace {

typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));

struct AttnArgs {
  const void* q;
  void* out;
  float* lse;
  const uint8_t *k_codes, *v_codes;
  const float *k_scale, *v_scale;
  const int32_t *cu, *table, *lens;
  int32_t* err;
  float *part_o, *part_ml;   // partial results of a split: rows of D floats, and (maximum, sum)
  int32_t* joins;            // dealt: the pair that each workgroup began and did not end (sequence, key head, parts)
  int64_t tokens, table_stride, num_pages, stride_t, stride_h;
  int32_t seqs, hq, hk, group, page_log2, table_width, max_q, causal, window;
  int32_t splits;            // of the keys of a (sequence, key head)
  int32_t workers;           // workgroups that the keys of all sequences are dealt to; 0: equal splits
  int32_t row_stride;        // rows of a partial result
  int32_t few_rows;          // sequences of at most so many rows are kv_attn_few_kernel's
  int32_t vec;               // q takes 16-byte loads
  float scale2;              // scale * log2(e)
};

constexpr float kInf = __builtin_inff();
constexpr float kLn2 = 0.69314718055994531f;

// Weights are exp2 of scores less a reference, which moves only where a weight would pass 2^8: sums and products lose nothing
// by that while the values are below 2^89, whatever the number of keys.  Where a page's scale is above kHugeScale (so that its
// values may reach 448 * 2^119), the reference lies 40 above the largest score from then on, and weights stay below 2^-32: 2^30
// keys of the largest value do not overflow, and only weights 2^-86 of the row's largest are lost.
constexpr float kHugeScale = 0x1p80f;
struct Reference {
  float room = 8.0f, lift = 0.0f;
  __device__ __forceinline__ void raise(bool huge) {  // the same for the whole wave
    if (huge) room = -32.0f, lift = 40.0f;
  }
};

// log sum_j exp(s_j) of a row whose weights 2^(s_j - m) have this sum.
__device__ __forceinline__ float row_lse(float m, float sum) {
  return ((m + (float)__builtin_amdgcn_frexp_expf(sum)) + __builtin_amdgcn_logf(__builtin_amdgcn_frexp_mantf(sum))) * kLn2;
}

// What a sequence's rows see.
struct Seq {
  int64_t row0;   // its first row of the batch
  int n, len;     // new tokens, length
  int lo, hi;     // keys that any of its rows may see, lo a multiple of 32
};

__device__ __forceinline__ bool seq_fits(const AttnArgs& a, int64_t c0, int64_t c1, int64_t len) {
  return c0 >= 0 && c1 <= a.tokens && c1 - c0 <= a.max_q && c1 - c0 <= len;
}

__device__ __forceinline__ void seq_keys(const AttnArgs& a, Seq& s) {
  const int64_t most = (int64_t)a.table_width << a.page_log2;
  s.hi = s.len < most ? s.len : (int)most;
  const int64_t first = (int64_t)s.len - s.n - a.window + 1;
  s.lo = a.window > 0 && first > 0 ? (int)first & ~31 : 0;
}

// False for a sequence without rows, and for one that does not fit (which sets the flag).
__device__ __forceinline__ bool seq_of(const AttnArgs& a, int b, Seq& s) {
  const int64_t c0 = a.cu[b], c1 = a.cu[b + 1], len = a.lens[b];
  if (c1 == c0) return false;
  if (c1 < c0 || !seq_fits(a, c0, c1, len)) {
    if (a.err) *a.err = 1;
    return false;
  }
  s.row0 = c0;
  s.n = (int)(c1 - c0);
  s.len = (int)len;
  if (len > (int64_t)a.table_width << a.page_log2 && a.err) *a.err = 1;
  seq_keys(a, s);
  return true;
}

// The keys [begin, end) of split x, and how many splits a span of keys takes: `splits` at most, each of a multiple
// of `unit` keys.
__device__ __forceinline__ int split_size(int span, int splits, int unit) {
  const int per = (span + splits - 1) / splits;
  return ((per + unit - 1) / unit) * unit;
}

// ---- conversions ----------------------------------------------------------------
template <int DT>
__device__ __forceinline__ uint32_t code_pair(uint32_t w, bool hi) {  // two codes of a dword as two operand elements
  if constexpr (DT == PDM_BF16) {
    return hi ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, true))
              : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, false));
  } else {
    return hi ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true))
              : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false));
  }
}
__device__ __forceinline__ uint32_t value_pair_lo(uint32_t w, float scale) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, false));
}
__device__ __forceinline__ uint32_t value_pair_hi(uint32_t w, float scale) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, true));
}

template <int DT>
__device__ __forceinline__ f32x4_t mfma16(u32x4_t a, u32x4_t b, f32x4_t c) {
  if constexpr (DT == PDM_BF16) return mfma16x16x32(a, b, c);
  else return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
}

// What rounding a pair of weights to the bf16 numbers `hi` left, as bf16 numbers.
__device__ __forceinline__ uint32_t remainder_pair(float x, float y, uint32_t hi) {
  return pack_bf16x2(x - __uint_as_float(hi << 16), y - __uint_as_float(hi & 0xffff0000u));
}

// A lane's value, for the whole wave.
__device__ __forceinline__ float lane_f(float v, int lane) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
}
__device__ __forceinline__ uint64_t lane_u64(uint64_t v, int lane) {
  return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32 |
         (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, lane);
}

// What is computed from x behind this is computed here: a rare branch stays one, where the compiler would have every call of
// the loop compute both sides.
__device__ __forceinline__ void only_here(uint32_t& x) { asm volatile("" : "+v"(x)); }

// NaN codes of a dword: bit 7 of each byte that holds one.
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }
// 0xff in the bytes whose bit 7 is set.
__device__ __forceinline__ uint32_t full_bytes(uint32_t n) { return (n << 1) - (n >> 7); }

template <int DT>
__device__ __forceinline__ void store4(void* base, int64_t at, float x, float y, float z, float w) {
  const u32x2_t v = DT == PDM_BF16 ? u32x2_t{pack_bf16x2(x, y), pack_bf16x2(z, w)}
                                   : u32x2_t{f32_to_f16_bits(x) | f32_to_f16_bits(y) << 16, f32_to_f16_bits(z) | f32_to_f16_bits(w) << 16};
  *reinterpret_cast<u32x2_t*>(static_cast<uint16_t*>(base) + at) = v;
}

__device__ __forceinline__ void store_out(const AttnArgs& a, int dt, int64_t at, float v) {
  static_cast<uint16_t*>(a.out)[at] = (uint16_t)(dt == PDM_BF16 ? f32_to_bf16_bits(v) : f32_to_f16_bits(v));
}

// Rows of the batch that no sequence covers, or one that does not fit: zeros.  One thread looks at a row, the
// block writes it.
template <int D>
__device__ __forceinline__ void clear_rows(const AttnArgs& a, int64_t first) {
  __shared__ int bad[256];
  const int64_t t = first + threadIdx.x;
  bool covered = false;
  if (t < a.tokens && a.seqs > 0) {
    int lo = 0, hi = a.seqs;  // last b with cu[b] <= t
    while (hi - lo > 1) {
      const int mid = lo + (hi - lo) / 2;
      if (a.cu[mid] <= t) lo = mid;
      else hi = mid;
    }
    const int64_t c0 = a.cu[lo], c1 = a.cu[lo + 1];
    covered = c0 <= t && t < c1 && seq_fits(a, c0, c1, a.lens[lo]);
  }
  bad[threadIdx.x] = t < a.tokens && !covered;
  if (!__syncthreads_or(t < a.tokens && !covered)) return;
  const int64_t left = a.tokens - first;
  const int rows = left < 256 ? (int)left : 256;
  for (int r = 0; r < rows; ++r) {
    if (!bad[r]) continue;
    u32x4_t* o = reinterpret_cast<u32x4_t*>(static_cast<uint16_t*>(a.out) + (first + r) * a.hq * D);
    for (int i = threadIdx.x; i < a.hq * D / 8; i += 256) o[i] = u32x4_t{0, 0, 0, 0};
    if (a.lse)
      for (int h = threadIdx.x; h < a.hq; h += 256) a.lse[(first + r) * a.hq + h] = -kInf;
  }
}

// ---- few rows ---------------------------------------------------------------------
// Up to 16 MT rows against a split of the keys.  Four waves take tiles of 32 keys in turn, each with its own
// maximum, sum and O, and join in LDS; splits join in kv_attn_join_kernel.  Bound by the bytes of the codes: a wave
// has the next tile's loads (8 KB at D = 128) in flight while it works on one; the operands come from registers, since no
// two waves share a key.  One token for 4 sequences of 60,000 to 120,000 tokens (32 query heads, 8 key heads of 128) 137 us,
// 5.2 TB/s, as fast as a copy; for 64 sequences of 128 to 8,192 65 us, 3.9 TB/s (59 and 5.4 for the join: what is missing is
// the first tile of each of 512 pairs and the run-out); 16 tokens for 256 sequences of 300 to 1,500 (6 heads of 64) 41 us,
// 3.8 TB/s; one token for one sequence of 1,000 9.6 us, two launches' latency.
constexpr int kFewKeys = 32, kFewWaves = 4, kFewStep = kFewKeys * kFewWaves;
constexpr int kDealt = 256;   // sequences of a call that is dealt

// What a workgroup works on: the keys [begin, end) of a (sequence, key head).
struct FewUnit {
  Seq sq;
  int b, kh, begin, end;
  bool alone;       // these are all keys of the pair
  int64_t slot;     // else the place of the partial result
};

__device__ __forceinline__ int steps_of(const Seq& s) { return s.hi > s.lo ? (s.hi - s.lo + kFewStep - 1) / kFewStep : 1; }

// Dealt: the steps of 128 keys of all (sequence, key head) pairs, in order, are dealt to `workers` workgroups in equal
// runs, so that a batch of long and short sequences keeps every CU busy to the end.  A run ends some pairs and begins
// one: a workgroup leaves at most two partial results, that of a pair which it did not begin (slot 2 w) and that of one which
// it did not end (2 w + 1).  Every workgroup computes the plan itself, a sequence per thread.  Against equal splits, 64
// sequences with 8 key heads of 128: of 128 to 8,192 tokens 63 us instead of 91, of 1,000 to 3,200 60 and 59 (these and those
// below before the weights' remainder, which costs all of them 1 to 2 %).
struct FewDeal {
  int64_t first[kDealt + 1];  // steps before a sequence, of all its heads
  int64_t sums[4];
  int most[4], some[4];       // steps of a wave's longest pair; its sequences that have any
  int row0[kDealt], n[kDealt], len[kDealt];
  int found;
};

// Where no pair has more than 1.25 times the average, every pair has workgroups of its own instead (`even`, equal parts of
// it): 64 sequences of 2,000 tokens 55 us instead of 61, of 1,700 to 2,300 56 instead of 61, 40 of 1,300 to 2,700 44 and 43.
__device__ __forceinline__ int64_t few_deal(const AttnArgs& a, FewDeal& sh, bool& even) {  // steps of a run
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  Seq s;
  int64_t steps = 0;
  if (tid < a.seqs && seq_of(a, tid, s) && (int64_t)s.n * a.group <= a.few_rows) {
    steps = (int64_t)steps_of(s) * a.hk;
    sh.row0[tid] = (int)s.row0, sh.n[tid] = s.n, sh.len[tid] = s.len;
  }
  int64_t upto = steps;
  for (int o = 1; o < 64; o <<= 1) {
    const int64_t v = __shfl_up(upto, o);
    upto += lane >= o ? v : 0;
  }
  const int most = (int)group_max((float)(steps / a.hk), 64);  // at most 2^23: exact
  const int some = __builtin_popcountll(__ballot(steps > 0));
  if (lane == 63) sh.sums[wave] = upto, sh.most[wave] = most, sh.some[wave] = some;
  __syncthreads();
  for (int w = 0; w < wave; ++w) upto += sh.sums[w];
  int top = 0, n = 0;
  for (int w = 0; w < 4; ++w) top = sh.most[w] > top ? sh.most[w] : top, n += sh.some[w];
  sh.first[tid] = upto - steps;
  if (tid == kDealt - 1) sh.first[kDealt] = upto;
  __syncthreads();
  const int64_t all = sh.first[kDealt];
  even = a.seqs * a.hk <= a.workers && (int64_t)top * n * a.hk * 4 <= all * 5;
  return (all + a.workers - 1) / a.workers;
}

// The part of run [x, to) that belongs to the pair at x; returns the steps taken.  FIRST: the run's first pair (a barrier);
// else u holds the pair before it.
template <bool FIRST>
__device__ __forceinline__ int64_t few_next(const AttnArgs& a, FewDeal& sh, int64_t x, int64_t from, int64_t to, int64_t worker,
                                            FewUnit& u) {
  if (FIRST) {
    if (sh.first[threadIdx.x] <= x && x < sh.first[threadIdx.x + 1]) sh.found = threadIdx.x;
    __syncthreads();
    u.b = __builtin_amdgcn_readfirstlane(sh.found);
  } else {
    while (sh.first[u.b + 1] <= x) ++u.b;  // x is below the last entry
  }
  u.sq.row0 = __builtin_amdgcn_readfirstlane(sh.row0[u.b]);
  u.sq.n = __builtin_amdgcn_readfirstlane(sh.n[u.b]);
  u.sq.len = __builtin_amdgcn_readfirstlane(sh.len[u.b]);
  seq_keys(a, u.sq);
  const int steps = steps_of(u.sq);
  const int64_t local = x - sh.first[u.b];
  u.kh = (int)(local / steps);
  const int s0 = (int)(local - (int64_t)u.kh * steps);
  const int n = to - x < steps - s0 ? (int)(to - x) : steps - s0;
  u.begin = u.sq.lo + s0 * kFewStep;
  u.end = s0 + n < steps ? u.begin + n * kFewStep : u.sq.hi;
  u.alone = n == steps;
  u.slot = 2 * worker + (x - s0 < from ? 0 : 1);
  return n;
}

// Not dealt: `splits` equal parts of each pair.
__device__ __forceinline__ bool few_split(const AttnArgs& a, int64_t unit, FewUnit& u) {
  const int split = (int)(unit % a.splits);
  const int64_t bh = unit / a.splits;
  u.kh = (int)(bh % a.hk), u.b = (int)(bh / a.hk);
  if (!seq_of(a, u.b, u.sq) || (int64_t)u.sq.n * a.group > a.few_rows) return false;
  const int size = split_size(u.sq.hi - u.sq.lo, a.splits, kFewStep);
  u.begin = u.sq.lo + split * size;
  if (split > 0 && u.begin >= u.sq.hi) return false;
  u.end = u.begin + size < u.sq.hi ? u.begin + size : u.sq.hi;
  u.alone = u.sq.hi - u.sq.lo <= size;
  u.slot = unit;
  return true;
}

template <int DT, int D, int MT>
__global__ void __launch_bounds__(256, D * MT <= 64 ? 4 : D * MT <= 128 ? 3 : D * MT <= 256 ? 2 : 1) kv_attn_few_kernel(AttnArgs a, int64_t units, int64_t guards) {
  constexpr int KK = D / 32;              // steps of the first product
  constexpr int DD = D / 16;              // tiles of the second: O^T row m of tile dd is element DD m + dd
  __shared__ float red[kFewWaves][16][D + 4];
  __shared__ float ml[kFewWaves + 1][2][16 * MT];
  __shared__ FewDeal deal;
  const int64_t unit = linear_block();
  if (unit >= units) {
    if (unit >= units + guards) return;
    const int64_t first = (unit - units) * 256;
    Seq s;
    // (sets the flag for a sequence that does not fit)
    if (units == 0 && first + threadIdx.x < a.seqs) seq_of(a, (int)first + threadIdx.x, s);
    clear_rows<D>(a, first);
    return;
  }
  int64_t x = 0, from = 0, to = 0;
  FewUnit fu;
  if (a.workers) {
    bool even;
    const int64_t per = few_deal(a, deal, even);
    int pair_parts = 0, pair_b = 0, pair_kh = 0;
    if (even) {
      const int shares = a.workers / (a.seqs * a.hk), i = (int)(unit % shares), pair = (int)(unit / shares);
      if (pair < a.seqs * a.hk) {
        pair_b = pair / a.hk, pair_kh = pair - pair_b * a.hk;
        const int steps = (int)((deal.first[pair_b + 1] - deal.first[pair_b]) / a.hk), size = (steps + shares - 1) / shares;
        const int64_t begin = deal.first[pair_b] + (int64_t)pair_kh * steps;
        if (i * size < steps) {
          from = begin + i * size;
          to = from + size < begin + steps ? from + size : begin + steps;
          pair_parts = i == 0 && size < steps ? (steps + size - 1) / size : 0;
        }
      }
    } else {
      from = unit * per;
      to = from + per < deal.first[kDealt] ? from + per : deal.first[kDealt];
    }
    x = from;
    if (threadIdx.x == 0) {
      int parts = 0;
      if (even) {
        parts = pair_parts;
        a.joins[4 * unit] = pair_b, a.joins[4 * unit + 1] = pair_kh;
      } else if (x < to && to < deal.first[kDealt]) {  // the pair of the last step, and where it ends
        int b = 0, n = kDealt;
        while (n > 1) {
          const int half = n >> 1;
          if (deal.first[b + half] < to) b += half, n -= half;
          else n = half;
        }
        Seq s;
        s.n = deal.n[b], s.len = deal.len[b];
        seq_keys(a, s);
        const int steps = steps_of(s);
        const int64_t kh = (to - 1 - deal.first[b]) / steps, begin = deal.first[b] + kh * steps;
        if (begin >= from && begin + steps > to) parts = (int)((begin + steps - 1) / per - unit) + 1;
        a.joins[4 * unit] = b, a.joins[4 * unit + 1] = (int)kh;
      }
      a.joins[4 * unit + 2] = parts;
    }
    if (x >= to) return;
  }
  if (a.workers) x += few_next<true>(a, deal, x, from, to, unit, fu);
  else if (!few_split(a, unit, fu)) return;

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4;
  u32x4_t q[MT][KK];                      // this lane's rows: queries, and the keys that they see
  int row_lo[MT], row_hi[MT];
  int all_lo, all_hi;                     // keys that every row sees (rows that are not there do not count)
  int kh, begin, end, mine;               // of the pair whose tiles are loaded; tiles of this wave
  const int32_t* table;
  // lane x of a batch of 32 tiles: place (in bytes) and scales of the 16 keys x % 2 of tile x / 2
  uint64_t spot = 0;
  float kss = 0.0f, vss = 0.0f;           // kss: NaN where the page does not exist
  Reference ref;
  auto key_of = [&](int i) { return begin + (wave + kFewWaves * i) * kFewKeys; };
  auto look_up = [&](int first) {
    const int key = key_of(first + (lane >> 1)) + (lane & 1) * 16;
    // (a page that does not exist: some page, its keys are not seen)
    spot = 0, kss = __builtin_nanf(""), vss = 0.0f;
    if (key < end) {
      const int id = table[key >> a.page_log2];
      if (id >= 0 && id < a.num_pages) {
        const int64_t entry = (int64_t)id * a.hk + kh;
        spot = (uint64_t)((entry << a.page_log2) + (key & ((1 << a.page_log2) - 1))) * D;
        kss = a.k_scale[entry];
        vss = a.v_scale[entry];
      } else if (a.err) {
        *a.err = 1;
      }
    }
    ref.raise(__any(vss > kHugeScale));
  };
  auto place = [&](int i, int s) { return lane_u64(spot, (i & 31) * 2 + s); };
  u32x4_t k[2][D / 64];                   // 16 bytes of a key row, 64 apart
  uint32_t v[2][4][D / 64];               // rows 4 g + i of 16 keys
  const uint32_t k_off = (uint32_t)(c * D + 16 * g);
  const uint32_t v_off = (uint32_t)(4 * g * D + (D / 16) * c);
  auto load_k = [&](int i) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const uint8_t* p = a.k_codes + place(i, s);
#pragma unroll
      for (int e = 0; e < D / 64; ++e) k[s][e] = *reinterpret_cast<const u32x4_t*>(p + k_off + 64 * e);
    }
  };
  auto load_v = [&](int i) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const uint8_t* p = a.v_codes + place(i, s);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        if constexpr (D == 64) {
          v[s][r][0] = *reinterpret_cast<const uint32_t*>(p + v_off + r * D);
        } else if constexpr (D == 128) {
          const u32x2_t w = *reinterpret_cast<const u32x2_t*>(p + v_off + r * D);
          v[s][r][0] = w[0], v[s][r][1] = w[1];
        } else {
          const u32x4_t w = *reinterpret_cast<const u32x4_t*>(p + v_off + r * D);
#pragma unroll
          for (int e = 0; e < 4; ++e) v[s][r][e] = w[e];
        }
      }
    }
  };
  // 4 x 4 bytes (keys x elements) of dword h of both halves, turned to pairs of keys: element tile x of it
  auto value_tile = [&](int h, int x, float s0, float s1) {
    const uint32_t sel = x < 2 ? 0x05010400u : 0x07030602u;
    const uint32_t w[4] = {__builtin_amdgcn_perm(v[0][1][h], v[0][0][h], sel), __builtin_amdgcn_perm(v[0][3][h], v[0][2][h], sel),
                           __builtin_amdgcn_perm(v[1][1][h], v[1][0][h], sel), __builtin_amdgcn_perm(v[1][3][h], v[1][2][h], sel)};
    return x & 1 ? u32x4_t{value_pair_hi(w[0], s0), value_pair_hi(w[1], s0), value_pair_hi(w[2], s1), value_pair_hi(w[3], s1)}
                 : u32x4_t{value_pair_lo(w[0], s0), value_pair_lo(w[1], s0), value_pair_lo(w[2], s1), value_pair_lo(w[3], s1)};
  };
  auto whole_tile = [&](int i, bool ok) { return ok && key_of(i) >= all_lo && key_of(i) + kFewKeys <= all_hi; };
  // What comes before a unit's first tile, and that tile's loads.
  auto start = [&]() {
    const Seq& sq = fu.sq;
    const int rows = sq.n * a.group;
    kh = fu.kh, begin = fu.begin, end = fu.end;
    table = a.table + (int64_t)fu.b * a.table_stride;
    int tiles = end > begin ? (end - begin + kFewKeys - 1) / kFewKeys : 0;
    if (tiles && a.num_pages == 0) {
      tiles = 0;
      if (a.err) *a.err = 1;
    }
    mine = tiles > wave ? (tiles - wave + kFewWaves - 1) / kFewWaves : 0;
    ref = Reference();
    if (mine > 0) look_up(0);
    all_lo = 0, all_hi = sq.hi;
    const int p0 = sq.len - sq.n, p1 = sq.len - 1;
    if (a.causal && p0 + 1 < all_hi) all_hi = p0 + 1;
    if (a.window > 0 && p1 - a.window + 1 > 0) all_lo = p1 - a.window + 1;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      const int r = mt * 16 + c;
      const int i = r / a.group, h = kh * a.group + (r - i * a.group);
      row_lo[mt] = 0x7fffffff, row_hi[mt] = 0;
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) q[mt][kk] = u32x4_t{0, 0, 0, 0};
      if (r < rows) {
        const int p = sq.len - sq.n + i;
        row_hi[mt] = a.causal && p + 1 < sq.hi ? p + 1 : sq.hi;
        row_lo[mt] = a.window > 0 && p - a.window + 1 > 0 ? p - a.window + 1 : 0;
        const uint16_t* y = static_cast<const uint16_t*>(a.q) + (sq.row0 + i) * a.stride_t + h * a.stride_h;
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) {
          const uint16_t* p8 = y + 64 * (kk >> 1) + 16 * g + 8 * (kk & 1);
          if (a.vec) {
            q[mt][kk] = *reinterpret_cast<const u32x4_t*>(p8);
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) q[mt][kk][e] = uint32_t(p8[2 * e]) | uint32_t(p8[2 * e + 1]) << 16;
          }
        }
      }
    }
    if (mine > 0) {
      load_k(0);
      load_v(0);
    }
  };
  start();

#pragma unroll 1
  for (;;) {
  float m[MT], l[MT];
  f32x4_t o[MT][DD];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    m[mt] = -kInf, l[mt] = 0.0f;
#pragma unroll
    for (int d = 0; d < DD; ++d) o[mt][d] = f32x4_t{0, 0, 0, 0};
  }
  // A NaN value must not reach rows that do not see its key (0 * NaN).  Where some row sees a tile in part, NaN codes are
  // taken out here and brought to the rows that see them after the loop.
  bool odd = false;
#pragma unroll 1
  for (int i = 0; i < mine; ++i) {
    const int x0 = (i & 31) * 2;
    const float ks[2] = {a.scale2 * lane_f(kss, x0), a.scale2 * lane_f(kss, x0 + 1)};
    const bool ok[2] = {ks[0] == ks[0], ks[1] == ks[1]};
    const float vs[2] = {lane_f(vss, x0), lane_f(vss, x0 + 1)};
    f32x4_t s[MT][2];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) s[mt][x] = f32x4_t{0, 0, 0, 0};
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) {
        const uint32_t w0 = k[x][kk >> 1][2 * (kk & 1)], w1 = k[x][kk >> 1][2 * (kk & 1) + 1];
        const u32x4_t kf = {code_pair<DT>(w0, false), code_pair<DT>(w0, true), code_pair<DT>(w1, false), code_pair<DT>(w1, true)};
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) s[mt][x] = mfma16<DT>(kf, q[mt][kk], s[mt][x]);
      }
    }
    if (i + 1 < mine) {
      if (((i + 1) & 31) == 0) look_up(i + 1);
      load_k(i + 1);
    }
    const int key = key_of(i);
    const bool whole = whole_tile(i, ok[0] && ok[1]);
    u32x4_t p[MT], rest[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      float w[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e] = s[mt][e >> 2][e & 3] * ks[e >> 2];
      if (!whole) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int j = key + 16 * (e >> 2) + 4 * g + (e & 3);
          w[e] = ok[e >> 2] && j >= row_lo[mt] && j < row_hi[mt] ? w[e] : -kInf;
        }
      }
      float top = w[0];
#pragma unroll
      for (int e = 1; e < 8; ++e) top = fmaxf(top, w[e]);
      if (__any(top > m[mt] + ref.room)) {
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
        const float now = top > m[mt] + ref.room ? top + ref.lift : m[mt];  // by row: other rows change nothing
        const float f = now == -kInf ? 1.0f : __builtin_amdgcn_exp2f(m[mt] - now);
        m[mt] = now;
        l[mt] *= f;
#pragma unroll
        for (int d = 0; d < DD; ++d) o[mt][d] *= f;
      }
      const float base = m[mt] == -kInf ? 0.0f : m[mt];
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e] = __builtin_amdgcn_exp2f(w[e] - base);
      l[mt] += ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        p[mt][e] = pack_bf16x2(w[2 * e], w[2 * e + 1]);
        rest[mt][e] = remainder_pair(w[2 * e], w[2 * e + 1], p[mt][e]);
      }
    }
    if (!whole) {
      uint32_t any = 0;
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int e = 0; e < D / 64; ++e) {
            const uint32_t n = nan_bytes(v[x][r][e]);
            any |= n;
            v[x][r][e] &= ~full_bytes(n);
          }
      odd = odd || __any(any != 0);
    }
#pragma unroll
    for (int h = 0; h < D / 64; ++h)
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const u32x4_t vf = value_tile(h, x, vs[0], vs[1]);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) o[mt][4 * h + x] = mfma16x16x32(vf, p[mt], mfma16x16x32(vf, rest[mt], o[mt][4 * h + x]));
      }
    if (i + 1 < mine) load_v(i + 1);
  }
  if (odd) {  // once more over the tiles that are seen in part: ones for NaN, ones for seen keys
#pragma unroll 1
    for (int i = 0; i < mine; ++i) {
      if ((i & 31) == 0) look_up(i);
      const float k0 = lane_f(kss, (i & 31) * 2), k1 = lane_f(kss, (i & 31) * 2 + 1);
      const bool ok[2] = {k0 == k0, k1 == k1};
      if (whole_tile(i, ok[0] && ok[1])) continue;
      load_v(i);
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int e = 0; e < D / 64; ++e) v[x][r][e] = (nan_bytes(v[x][r][e]) >> 7) * 0x38u;  // the code of 1
      u32x4_t seen[MT];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int j = key_of(i) + 16 * (e >> 1) + 4 * g + 2 * (e & 1);
          seen[mt][e] = (ok[e >> 1] && j >= row_lo[mt] && j < row_hi[mt] ? 0x3f80u : 0u) |
                        (ok[e >> 1] && j + 1 >= row_lo[mt] && j + 1 < row_hi[mt] ? 0x3f800000u : 0u);
        }
#pragma unroll
      for (int h = 0; h < D / 64; ++h)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const u32x4_t ones = value_tile(h, x, 1.0f, 1.0f);
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            const f32x4_t hits = mfma16x16x32(ones, seen[mt], f32x4_t{0, 0, 0, 0});
#pragma unroll
            for (int e = 0; e < 4; ++e) o[mt][4 * h + x][e] += hits[e] > 0.0f ? __builtin_nanf("") : 0.0f;
          }
        }
    }
  }

  // the next pair's first loads are in flight while this one's waves join
  const FewUnit cur = fu;
  const int rows = cur.sq.n * a.group;
  const bool more = x < to;
  if (more) {
    x += few_next<false>(a, deal, x, from, to, unit, fu);
    start();
  }
  // the sums of a row are spread over its four lanes
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    l[mt] += __shfl_xor(l[mt], 16);
    l[mt] += __shfl_xor(l[mt], 32);
    if (g == 0) {
      ml[wave][0][mt * 16 + c] = m[mt];
      ml[wave][1][mt * 16 + c] = l[mt];
    }
  }
  lds_barrier();
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    const int r = mt * 16 + c;
    float top = ml[0][0][r];
#pragma unroll
    for (int w = 1; w < kFewWaves; ++w) top = fmaxf(top, ml[w][0][r]);
    const float f = m[mt] == -kInf ? (l[mt] != l[mt] ? 1.0f : 0.0f) : __builtin_amdgcn_exp2f(m[mt] - top);
    if (wave == 0 && g == 0) {  // maximum and sum of the row
      float sum = 0.0f;
#pragma unroll
      for (int w = 0; w < kFewWaves; ++w)
        sum += ml[w][1][r] * (ml[w][0][r] == -kInf ? 1.0f : __builtin_amdgcn_exp2f(ml[w][0][r] - top));
      ml[kFewWaves][0][r] = top, ml[kFewWaves][1][r] = sum;
    }
    if (mt) lds_barrier();
    if (r < rows) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int d = 0; d < DD; d += 4)
          *reinterpret_cast<f32x4_t*>(&red[wave][c][DD * (4 * g + e) + d]) =
              f32x4_t{o[mt][d][e] * f, o[mt][d + 1][e] * f, o[mt][d + 2][e] * f, o[mt][d + 3][e] * f};
    }
    lds_barrier();
    const int here = rows - mt * 16 < 16 ? rows - mt * 16 : 16;
    for (int i4 = threadIdx.x; i4 < here * (D / 4); i4 += 256) {
      const int rr = i4 / (D / 4), d = 4 * (i4 - rr * (D / 4)), row = mt * 16 + rr;
      f32x4_t acc = {0, 0, 0, 0};
#pragma unroll
      for (int w = 0; w < kFewWaves; ++w) acc += *reinterpret_cast<const f32x4_t*>(&red[w][rr][d]);
      const float top_r = ml[kFewWaves][0][row], sum = ml[kFewWaves][1][row];
      if (cur.alone) {
        const int i = row / a.group, h = cur.kh * a.group + (row - i * a.group);
        const int64_t at = (cur.sq.row0 + i) * a.hq + h;
        const float inv = sum != 0.0f ? 1.0f / sum : 0.0f;
        store4<DT>(a.out, at * D + d, acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv);
        if (d == 0 && a.lse) a.lse[at] = sum != 0.0f ? row_lse(top_r, sum) : -kInf;
      } else {
        const int64_t at = cur.slot * a.row_stride + row;
        *reinterpret_cast<f32x4_t*>(a.part_o + at * D + d) = acc;
        if (d == 0) {
          a.part_ml[2 * at] = top_r;
          a.part_ml[2 * at + 1] = sum;
        }
      }
    }
  }
  if (!more) return;
  lds_barrier();
  }
}

// Joins the `used` partial results of one row, in the workspace rows at(0 .. used - 1), in a wave (W = 1) or by the W waves of
// a block.  A lane holds the maximum and sum of one split, so that only the rows of O are read one after the other.
template <int DT, int D, int W, typename F>
__device__ __forceinline__ void join_row(const AttnArgs& a, int used, int64_t out, F at) {
  constexpr int E = D / 64;
  __shared__ float part[W][D + 1];
  __shared__ float tops[W];
  const int lane = threadIdx.x & 63, wave = W == 1 ? 0 : threadIdx.x >> 6;
  const int s0 = (int)((int64_t)used * wave / W), s1 = (int)((int64_t)used * (wave + 1) / W);
  float top = -kInf, sum = 0.0f, acc[E];
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = 0.0f;
  for (int base = s0; base < s1; base += 64) {
    float m = -kInf, l = 0.0f;
    if (base + lane < s1) {
      const int64_t pr = at(base + lane);
      m = a.part_ml[2 * pr], l = a.part_ml[2 * pr + 1];
    }
    const float now = fmaxf(top, group_max(m, 64));
    const float back = top == -kInf ? 1.0f : __builtin_amdgcn_exp2f(top - now);
    const float f = m == -kInf ? (l != l ? 1.0f : 0.0f) : __builtin_amdgcn_exp2f(m - now);
    sum = sum * back + group_sum(l * f, 64);
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] *= back;
    top = now;
    const int n = s1 - base < 64 ? s1 - base : 64;
#pragma unroll 8
    for (int s = 0; s < n; ++s) {
      const float fs = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, f), s));
      const float* o = a.part_o + at(base + s) * D + lane * E;
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] = __builtin_fmaf(o[e], fs, acc[e]);
    }
  }
  if constexpr (W > 1) {
    if (lane == 0) tops[wave] = top;
    __syncthreads();
    float all = tops[0];
#pragma unroll
    for (int w = 1; w < W; ++w) all = fmaxf(all, tops[w]);
    const float f = top == -kInf ? (sum != sum ? 1.0f : 0.0f) : __builtin_amdgcn_exp2f(top - all);
#pragma unroll
    for (int e = 0; e < E; ++e) part[wave][lane * E + e] = acc[e] * f;
    if (lane == 0) part[wave][D] = sum * f;
    __syncthreads();
    if (wave) return;
    sum = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = 0.0f;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      sum += part[w][D];
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] += part[w][lane * E + e];
    }
    top = all;
  }
#pragma unroll
  for (int e = 0; e < E; ++e) store_out(a, DT, out * D + lane * E + e, sum != 0.0f ? acc[e] / sum : 0.0f);
  if (lane == 0 && a.lse) a.lse[out] = sum != 0.0f ? row_lse(top, sum) : -kInf;
}

// Joins the equal parts of the few-rows kernel's pairs: W waves per row.
template <int DT, int D, int W>
__global__ void __launch_bounds__(256) kv_attn_join_kernel(AttnArgs a, int64_t units) {
  const int64_t x = W == 1 ? linear_block() * 4 + (threadIdx.x >> 6) : linear_block();
  if (x >= units) return;
  const int row = (int)(x % a.row_stride);
  const int64_t bh = x / a.row_stride;
  const int kh = (int)(bh % a.hk), b = (int)(bh / a.hk);
  Seq sq;
  if (!seq_of(a, b, sq)) return;
  const int64_t rows = (int64_t)sq.n * a.group;
  if (rows > a.few_rows || row >= rows) return;
  const int size = split_size(sq.hi - sq.lo, a.splits, kFewStep);
  const int used = sq.hi > sq.lo ? (sq.hi - sq.lo + size - 1) / size : 1;
  if (used == 1) return;
  const int i = row / a.group, h = kh * a.group + (row - i * a.group);
  join_row<DT, D, W>(a, used, (sq.row0 + i) * a.hq + h, [&](int s) { return (bh * a.splits + s) * a.row_stride + row; });
}

// Joins the dealt pairs: a workgroup for each that began a pair and did not end it, a wave per row in turn.
template <int DT, int D>
__global__ void __launch_bounds__(256) kv_attn_dealt_join_kernel(AttnArgs a) {
  const int64_t w = blockIdx.x;
  const int parts = a.joins[4 * w + 2];
  if (parts < 2) return;
  const int b = a.joins[4 * w], kh = a.joins[4 * w + 1];
  const int64_t row0 = a.cu[b];
  const int rows = (int)(a.cu[b + 1] - row0) * a.group;
  for (int row = threadIdx.x >> 6; row < rows; row += 4) {
    const int i = row / a.group, h = kh * a.group + (row - i * a.group);
    join_row<DT, D, 1>(a, parts, (row0 + i) * a.hq + h, [&](int s) { return (2 * (w + s) + (s == 0)) * a.row_stride + row; });
  }
}

// ---- many rows ---------------------------------------------------------------------
// 128 NG rows of a (sequence, key head) against its keys, NG groups of four waves of 32 rows.  A wave takes tiles of KT
// keys in two phases: products (O += V^T P of the tile before, S of this one) and softmax (P from S), with a barrier
// after each.  With two groups the second is one phase behind the first, so that on every SIMD a wave's products run
// beside the other's softmax; left to themselves, two waves of a SIMD were found in the same phase and took turns.
// Tiles are converted once on their way into LDS, in the softmax phase, their loads a phase earlier: K as rows by the
// first group, V transposed by the second, its keys in the order in which the first product leaves P.
// Bound by the softmax phase: two prompts of 3,500 to 4,500 tokens behind 3,000 to 5,000 (32 query heads, 8 key heads of 128)
// 786 to 809 us by the card, 0.96 to 0.98 PFLOP/s, where a bf16 product of 8,192^3 reaches 1.37.  The matrix units are busy
// 44 % of the time and the vector units as long; a tile's products take 1,024 cycles of a wave at best, its softmax about 1,400
// (512 of them exponentials) and staging 500.  Tried on it: loads in the softmax phase (854 us against 796), staging between
// the products (857 against 834), priority for either phase (no change or 3 % slower).
template <int D, int KT>
struct ManyShared {
  static constexpr int KS = 2 * D + 16;    // bytes of a K row: 16 rows of a fragment read fall into different banks
  static constexpr int VS = 2 * KT;        // bytes of a V^T row, its 16-byte pieces exchanged by turn()
  // Piece g of row d lies at g ^ turn(d): any 16 rows of a fragment read, and the 8 rows that 8 lanes write at a time
  // (rows 16 apart), fall into different banks.  (With rows padded to 144 bytes a write took 32 cycles instead of 8.)
  __device__ static constexpr int turn(int d) { return KT == 64 ? ((d >> 1) ^ (d >> 4)) & 7 : ((d >> 2) ^ (d >> 4)) & 3; }
  alignas(16) char k[2][KT * KS];
  alignas(16) char v[2][D * VS];
  float sc[2][KT / 16];                    // scale2 * scale of 16 keys; NaN where their page does not exist
  int odd[8];                              // a wave's share of V held NaN
};

// Block `item` of the list of (sequence, M rows): sequence b's span begins at cu[b] * group / M + b.
template <int M>
__device__ __forceinline__ bool many_block(const AttnArgs& a, int64_t item, Seq& sq, int& b, int& r0) {
  b = find_sequence(a.seqs, item, [&](int i) { return (int64_t)a.cu[i] * a.group / M + i; });
  const int64_t j = item - ((int64_t)a.cu[b] * a.group / M + b);
  if (j < 0 || !seq_of(a, b, sq)) return false;
  const int64_t rows = (int64_t)sq.n * a.group;
  if (rows <= a.few_rows || j * M >= rows) return false;
  r0 = (int)(j * M);
  return true;
}

// The keys that rows r0 .. r0 + M - 1 may see: [lo, hi), lo a multiple of 32.
template <int M>
__device__ __forceinline__ void many_keys(const AttnArgs& a, const Seq& sq, int r0, int& lo, int& hi) {
  const int rows = sq.n * a.group;
  const int i0 = r0 / a.group, i1 = ((r0 + M < rows ? r0 + M : rows) - 1) / a.group;
  const int p0 = sq.len - sq.n + i0, p1 = sq.len - sq.n + i1;
  hi = a.causal && p1 + 1 < sq.hi ? p1 + 1 : sq.hi;
  lo = a.window > 0 && p0 - a.window + 1 > 0 ? (p0 - a.window + 1) & ~31 : 0;
  if (lo > hi) lo = hi & ~31;
}

template <int DT>
__device__ __forceinline__ f32x16_t mfma32(u32x4_t a, u32x4_t b, f32x16_t c) {
  if constexpr (DT == PDM_BF16) return mfma32x32x16(a, b, c);
  else return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
}

template <int DT, int D, int KT, int NG>
__global__ void __launch_bounds__(256 * NG, D == 256 ? 1 : 2) kv_attn_many_kernel(AttnArgs a, int64_t items) {
  constexpr int M = 128 * NG;
  constexpr int KK = D / 16, DD = D / 32, XX = KT / 32;
  constexpr int KP = KT * D / 16 / 256;    // 16-byte pieces of a K tile per thread
  constexpr int VD = D == 64 ? 4 : 8;      // elements of a thread's 4 keys of V
  constexpr int KS = ManyShared<D, KT>::KS, VS = ManyShared<D, KT>::VS;
  constexpr int LEAD = 8;                  // fragments read ahead of their products
  constexpr bool FINE = DT == PDM_F16;     // weights as two bf16 numbers (see the head of the file)
  __shared__ ManyShared<D, KT> sh;

  const int64_t unit = linear_block();
  const int split = (int)(unit % a.splits);
  const int64_t ih = unit / a.splits;
  const int kh = (int)(ih % a.hk);
  const int64_t item = items - 1 - ih / a.hk;  // later rows see more keys: they begin first
  if (item < 0) return;
  Seq sq;
  int b, r0;
  if (!many_block<M>(a, item, sq, b, r0)) return;
  int lo, hi;
  many_keys<M>(a, sq, r0, lo, hi);
  const int size = split_size(hi - lo, a.splits, KT);
  const int begin = lo + split * size;
  if (split > 0 && begin >= hi) return;
  const int end = begin + size < hi ? begin + size : hi;
  const int rows = sq.n * a.group;
  int tiles = end > begin ? (end - begin + KT - 1) / KT : 0;
  if (tiles && a.num_pages == 0) {
    tiles = 0;
    if (a.err) *a.err = 1;
  }

  const int tid = threadIdx.x & 255, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);  // of the group
  const int grp = NG == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 8);
  const int c = lane & 31, h = lane >> 5;

  // this lane's row: its query, and the keys that it sees
  u32x4_t q[KK];
  int row_lo = 0x7fffffff, row_hi = 0;
  const int row = r0 + grp * 128 + wave * 32 + c;
  const int tok = row / a.group, head = kh * a.group + (row - tok * a.group);
#pragma unroll
  for (int kk = 0; kk < KK; ++kk) q[kk] = u32x4_t{0, 0, 0, 0};
  if (row < rows) {
    const int p = sq.len - sq.n + tok;
    row_hi = a.causal && p + 1 < sq.hi ? p + 1 : sq.hi;
    row_lo = a.window > 0 && p - a.window + 1 > 0 ? p - a.window + 1 : 0;
    const uint16_t* x = static_cast<const uint16_t*>(a.q) + (sq.row0 + tok) * a.stride_t + head * a.stride_h + 8 * h;
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
      if (a.vec) {
        q[kk] = *reinterpret_cast<const u32x4_t*>(x + 16 * kk);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) q[kk][e] = uint32_t(x[16 * kk + 2 * e]) | uint32_t(x[16 * kk + 2 * e + 1]) << 16;
      }
    }
  }
  if (a.scale2 < 0.0f) {  // the scale's sign goes into the queries
#pragma unroll
    for (int kk = 0; kk < KK; ++kk)
#pragma unroll
      for (int e = 0; e < 4; ++e) q[kk][e] ^= 0x80008000u;
  }
  // keys that every row of this wave sees
  int all_lo = 0, all_hi = sq.hi;
  {
    const int w0 = r0 + grp * 128 + wave * 32;
    if (w0 < rows) {
      const int w1 = (w0 + 32 < rows ? w0 + 32 : rows) - 1;
      const int p0 = sq.len - sq.n + w0 / a.group, p1 = sq.len - sq.n + w1 / a.group;
      if (a.causal && p0 + 1 < all_hi) all_hi = p0 + 1;
      if (a.window > 0 && p1 - a.window + 1 > 0) all_lo = p1 - a.window + 1;
    }
  }

  // ---- staging ----
  const int32_t* table = a.table + (int64_t)b * a.table_stride;
  const int mask = (1 << a.page_log2) - 1;
  constexpr int PER = 1024 / KT;           // tiles of a batch of 1024 keys
  uint64_t spot = 0;                       // lane i: place and scales of keys 16 i .. of the batch
  float kss = 0.0f, vss = 0.0f;
  Reference ref;
  u32x4_t kr[KP];
  u32x4_t vw[D == 64 ? 1 : 2];             // 16 elements of a key, or of two keys
  uint32_t vr[4][VD / 4];                  // VD elements of four keys, exchanged
  float v_scale = 0.0f;
  const int kc = (tid % (D / 16)) * 16, kr0 = tid / (D / 16);       // piece and row of K, 4096 / D rows a pass
  // V: lanes 0 .. 31 and 32 .. 63 (D = 64: a row of 16 lanes each) load keys of the same four, 16 elements of each, and
  // then exchange them for VD elements of all four: piece vm, four keys va
  constexpr int VC = D / 16;               // 16-byte pieces of a row
  const int va = D == 256 ? wave * 2 + (lane >> 4 & 1) : wave * 4 + (D == 64 ? lane >> 2 & 3 : lane >> 3 & 3);
  const int vm = D == 64 ? 4 * (lane & 3) + (lane >> 4) : 2 * (lane & (VC - 1)) + (lane >> 5);
  uint32_t k_off[KP];
#pragma unroll
  for (int p = 0; p < KP; ++p) k_off[p] = ((kr0 + p * (4096 / D)) & 15) * D + kc;
  const uint32_t v_off = ((va & 3) * 4 + (D == 64 ? lane >> 4 : 2 * (lane >> 5))) * D + 16 * (lane & (VC - 1));
  // KV: 1 K, 2 V, 3 both (a type's value)
  auto load = [&](int t, auto kv) {
    const int key0 = begin + t * KT;
    if (t % PER == 0) {
      const int key = key0 + 16 * lane;
      // (a page that does not exist: some page, its keys are not seen)
      spot = 0, kss = __builtin_nanf(""), vss = 0.0f;
      if (key < end) {
        const int id = table[key >> a.page_log2];
        if (id >= 0 && id < a.num_pages) {
          const int64_t entry = (int64_t)id * a.hk + kh;
          spot = (uint64_t)((entry << a.page_log2) + (key & mask)) * D;
          // not zero: a hidden score times it stays -inf
          kss = fmaxf(a.k_scale[entry] * fabsf(a.scale2), 0x1p-126f);
          vss = a.v_scale[entry];
        } else if (a.err) {
          *a.err = 1;
        }
      }
      ref.raise(__any(vss > kHugeScale));
    }
    const int g0 = (t % PER) * (KT / 16);
    auto place = [&](int grp) { return lane_u64(spot, g0 + grp); };  // bytes before the 16 keys `grp` of the tile
    if constexpr (decltype(kv)::value & 1) {
#pragma unroll
      for (int p = 0; p < KP; ++p) {
        const int grp = __builtin_amdgcn_readfirstlane((kr0 + p * (4096 / D)) >> 4);
        kr[p] = *reinterpret_cast<const u32x4_t*>(a.k_codes + place(grp) + k_off[p]);
      }
    }
    if constexpr (decltype(kv)::value & 2) {
      const int grp = D == 256 ? wave >> 1 : wave;
      v_scale = lane_f(vss, g0 + grp);
      const uint8_t* p = a.v_codes + place(grp) + v_off;
#pragma unroll
      for (int r = 0; r < (D == 64 ? 1 : 2); ++r) vw[r] = *reinterpret_cast<const u32x4_t*>(p + r * D);
    }
  };
  auto exchange = [&]() {
    if constexpr (D == 64) {
      const u32x2_t x = __builtin_amdgcn_permlane32_swap(vw[0][0], vw[0][2], false, false);
      const u32x2_t y = __builtin_amdgcn_permlane32_swap(vw[0][1], vw[0][3], false, false);
      const u32x2_t lo = __builtin_amdgcn_permlane16_swap(x[0], y[0], false, false);
      const u32x2_t hi = __builtin_amdgcn_permlane16_swap(x[1], y[1], false, false);
      vr[0][0] = lo[0], vr[1][0] = lo[1], vr[2][0] = hi[0], vr[3][0] = hi[1];
    } else {
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const u32x2_t x = __builtin_amdgcn_permlane32_swap(vw[r][e], vw[r][2 + e], false, false);
          vr[r][e] = x[0], vr[2 + r][e] = x[1];
        }
    }
  };
  // the K scales of tile t: the lanes that hold them (before the next batch is looked up)
  auto stage_sc = [&](int t) {
    const uint32_t x = lane - (t % PER) * (KT / 16);
    if (wave == 0 && x < KT / 16) sh.sc[t & 1][x] = kss;
  };
  auto stage_k = [&](int t) {
    char* kb = sh.k[t & 1];
#pragma unroll
    for (int p = 0; p < KP; ++p) {
      char* dst = kb + (kr0 + p * (4096 / D)) * KS + 2 * kc;
      u32x4_t w0, w1;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        w0[2 * e] = code_pair<DT>(kr[p][e], false), w0[2 * e + 1] = code_pair<DT>(kr[p][e], true);
        w1[2 * e] = code_pair<DT>(kr[p][2 + e], false), w1[2 * e + 1] = code_pair<DT>(kr[p][2 + e], true);
      }
      *reinterpret_cast<u32x4_t*>(dst) = w0;
      *reinterpret_cast<u32x4_t*>(dst + 16) = w1;
    }
    stage_sc(t);
  };
  // V^T of tile t; NaN codes become zeros here (0 * NaN would reach rows that do not see the key) and are remembered, or,
  // in MARK, ones where everything else becomes zero.
  bool odd = false;
  auto stage_v = [&](int t, auto mark) {
    // keys 4 va .. + 3: block va % 4 of their 16; blocks 0, 2 belong to lanes h = 0 of the product, 1, 3 to h = 1
    const int x = va & 3;
    const uint32_t at = vm * VD * VS + 16 * ((2 * (va >> 2) + (x & 1)) ^ ManyShared<D, KT>::turn(vm * VD)) + 8 * (x >> 1);
    exchange();
    uint32_t nan = 0;
#pragma unroll
    for (int e = 0; e < VD / 4; ++e)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const uint32_t n = nan_bytes(vr[r][e]);
        nan |= n;
        if constexpr (decltype(mark)::value) vr[r][e] = (n >> 7) * 0x38u;  // 0x38: the code of 1
      }
    if constexpr (!decltype(mark)::value) {
      if (__any(nan != 0)) {
        odd = true;
#pragma unroll
        for (int e = 0; e < VD / 4; ++e)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            only_here(vr[r][e]);
            vr[r][e] &= ~full_bytes(nan_bytes(vr[r][e]));
          }
      }
    }
    const float f = decltype(mark)::value ? 1.0f : v_scale;
#pragma unroll
    for (int e = 0; e < VD / 4; ++e) {
      const uint32_t w01[2] = {__builtin_amdgcn_perm(vr[1][e], vr[0][e], 0x05010400u), __builtin_amdgcn_perm(vr[1][e], vr[0][e], 0x07030602u)};
      const uint32_t w23[2] = {__builtin_amdgcn_perm(vr[3][e], vr[2][e], 0x05010400u), __builtin_amdgcn_perm(vr[3][e], vr[2][e], 0x07030602u)};
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        const u32x2_t w = d & 1 ? u32x2_t{value_pair_hi(w01[d >> 1], f), value_pair_hi(w23[d >> 1], f)}
                                : u32x2_t{value_pair_lo(w01[d >> 1], f), value_pair_lo(w23[d >> 1], f)};
        const int r = 4 * e + d;  // turn(row + r) = turn(row) ^ turn(r) for the 4 or 8 rows of a thread
        *reinterpret_cast<u32x2_t*>(sh.v[t & 1] + (at ^ (16 * ManyShared<D, KT>::turn(r))) + r * VS) = w;
      }
    }
  };

  // ---- products ----
  float m = -kInf, l = 0.0f;
  f32x16_t o[DD], s[XX];
  constexpr f32x16_t zero16 = {0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
  for (int d = 0; d < DD; ++d) o[d] = zero16;
  const uint32_t k_at = c * KS + 16 * h;
  const uint32_t v_at = c * VS + 16 * (h ^ ManyShared<D, KT>::turn(c));
  // V^T fragment of rows 32 d + c and keys 16 y ..
  auto v_frag = [&](int t, int d, int y) {
    return *reinterpret_cast<const u32x4_t*>(sh.v[t & 1] + (v_at ^ (32 * y ^ 16 * ManyShared<D, KT>::turn(32 * d))) + d * 32 * VS);
  };
  // s = scores of tile t (products alone)
  auto scores = [&](int t) {
    const char* kb = sh.k[t & 1] + k_at;
#pragma unroll
    for (int x = 0; x < XX; ++x) s[x] = zero16;
#pragma unroll
    for (int kk = 0; kk < KK; ++kk)
#pragma unroll
      for (int x = 0; x < XX; ++x)
        s[x] = mfma32<DT>(*reinterpret_cast<const u32x4_t*>(kb + x * 32 * KS + 32 * kk), q[kk], s[x]);
    sched_mfma_ds_pipeline<XX * KK, LEAD>();
  };
  // the running maximum, and P from the scores
  u32x4_t p[2 * XX], rest[2 * XX];
  auto weights = [&](int t) __attribute__((always_inline)) {
    const int key = begin + t * KT;
    float sc[2 * XX];                      // of 16 keys each, not negative
    bool ok = true;
#pragma unroll
    for (int x = 0; x < 2 * XX; ++x) {
      sc[x] = __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, sh.sc[t & 1][x])));
      ok = ok && sc[x] == sc[x];
    }
    if (!(key >= all_lo && key + KT <= all_hi)) {
      uint32_t from = key + 4 * h - row_lo, span = row_hi > row_lo ? row_hi - row_lo : 0;  // seen: j - row_lo < span
      only_here(from);
#pragma unroll
      for (int x = 0; x < XX; ++x)
#pragma unroll
        for (int e = 0; e < 16; ++e) s[x][e] = from + (32 * x + 8 * (e >> 2) + (e & 3)) < span ? s[x][e] : -kInf;
    }
    if (!ok) {
#pragma unroll
      for (int x = 0; x < 2 * XX; ++x)
        if (sc[x] != sc[x]) {
          sc[x] = 1.0f;
#pragma unroll
          for (int e = 0; e < 8; ++e) s[x >> 1][8 * (x & 1) + e] = -kInf;
        }
    }
    float top = -kInf;
#pragma unroll
    for (int x = 0; x < 2 * XX; ++x) {
      float most = s[x >> 1][8 * (x & 1)];
#pragma unroll
      for (int e = 1; e < 8; ++e) most = fmaxf(most, s[x >> 1][8 * (x & 1) + e]);
      top = fmaxf(top, most * sc[x]);
    }
    if (__any(top > m + ref.room)) {
      top = fmaxf(top, __shfl_xor(top, 32));
      const float now = top > m + ref.room ? top + ref.lift : m;  // by row: other rows change nothing
      const float f = now == -kInf ? 1.0f : __builtin_amdgcn_exp2f(m - now);
      m = now;
      l *= f;
#pragma unroll
      for (int d = 0; d < DD; ++d) o[d] *= f;
    }
    const float base = m == -kInf ? 0.0f : m;
#pragma unroll
    for (int x = 0; x < XX; ++x) {
      float v[16];
#pragma unroll
      for (int e = 0; e < 16; ++e) v[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[x][e], sc[2 * x + (e >> 3)], -base));
#pragma unroll
      for (int e = 0; e < 16; e += 4) l += (v[e] + v[e + 1]) + (v[e + 2] + v[e + 3]);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        p[2 * x][e] = pack_bf16x2(v[2 * e], v[2 * e + 1]);
        p[2 * x + 1][e] = pack_bf16x2(v[8 + 2 * e], v[8 + 2 * e + 1]);
        if constexpr (FINE) {
          rest[2 * x][e] = remainder_pair(v[2 * e], v[2 * e + 1], p[2 * x][e]);
          rest[2 * x + 1][e] = remainder_pair(v[8 + 2 * e], v[8 + 2 * e + 1], p[2 * x + 1][e]);
        }
      }
    }
  };
  auto values = [&](int t) __attribute__((always_inline)) {  // (not inlined, it would have O in memory)
#pragma unroll
    for (int y = 0; y < 2 * XX; ++y) {
      u32x4_t vf[DD];
#pragma unroll
      for (int d = 0; d < DD; ++d) {
        vf[d] = v_frag(t, d, y);
        o[d] = mfma32x32x16(vf[d], p[y], o[d]);
      }
      if constexpr (FINE) {
#pragma unroll
        for (int d = 0; d < DD; ++d) o[d] = mfma32x32x16(vf[d], rest[y], o[d]);
      }
    }
    sched_mfma_ds_pipeline<2 * XX * DD, LEAD, FINE ? 2 : 1>();
  };

  if (tiles > 0) {
    // Barrier k + 1 begins phase k: the first group has products at even ones, the second at odd ones.  K of tile t + 1 is
    // written in phase 2 t + 1, where the other group reads that of tile t; V of tile t + 1 in phase 2 t + 2 (or before the
    // barrier between them, where there is one group): what either overwrites was last read in an earlier phase.  Behind
    // the last tile that one is loaded and written again, to no use.  V is written behind the weights: its loads have most
    // of two phases, and its writes come when the other group reads its last fragments (880 us -> 843 for two prompts of
    // 4,000 tokens behind 4,000; keys behind the weights too: 854).
    auto run = [&](auto kv) {
      auto keys = [&](int t) {
        if constexpr (decltype(kv)::value & 1) stage_k(t);
      };
      auto vals = [&](int t) {
        if constexpr (decltype(kv)::value & 2) stage_v(t, std::false_type());
      };
      const int last = tiles - 1;
      load(0, kv);
      keys(0);
      vals(0);
      if (decltype(kv)::value == 2) lds_barrier();
      lds_barrier();
      load(last > 0 ? 1 : 0, kv);
      scores(0);
      lds_barrier();
      keys(1);
      weights(0);
      vals(1);
#pragma unroll 1
      for (int t = 1; t < tiles; ++t) {
        lds_barrier();
        load(last < t + 1 ? last : t + 1, kv);
        __builtin_amdgcn_sched_barrier(0);
        values(t - 1);
        __builtin_amdgcn_sched_barrier(0);
        scores(t);
        __builtin_amdgcn_sched_barrier(0);
        lds_barrier();
        __builtin_amdgcn_sched_barrier(0);
        keys(t + 1);
        __builtin_amdgcn_sched_barrier(0);
        weights(t);
        __builtin_amdgcn_sched_barrier(0);
        vals(t + 1);
      }
      lds_barrier();
      values(last);
      if (decltype(kv)::value == 1) lds_barrier();
    };
    if (NG == 1) run(std::integral_constant<int, 3>());
    else if (grp == 0) run(std::integral_constant<int, 1>());
    else run(std::integral_constant<int, 2>());

    // NaN among the values of any wave's share: once more over the tiles, with ones for NaN and for keys that are seen
    if (lane == 0) sh.odd[grp * 4 + wave] = odd;
    lds_barrier();
    int any = 0;
#pragma unroll
    for (int w = 0; w < 4 * NG; ++w) any |= sh.odd[w];
    if (any) {
#pragma unroll 1
      for (int t = 0; t < tiles; ++t) {
        load(t, std::integral_constant<int, 2>());
        lds_barrier();  // the tile before is done with
        if (grp == NG - 1) {
          stage_v(t, std::true_type());
          stage_sc(t);
        }
        lds_barrier();
#pragma unroll 1
        for (int y = 0; y < 2 * XX; ++y) {
          u32x4_t seen;
          const bool ok = sh.sc[t & 1][y] == sh.sc[t & 1][y];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int j = begin + t * KT + 16 * y + 8 * (e >> 1) + 4 * h + 2 * (e & 1);
            seen[e] = (ok && j >= row_lo && j < row_hi ? 0x3f80u : 0u) | (ok && j + 1 >= row_lo && j + 1 < row_hi ? 0x3f800000u : 0u);
          }
#pragma unroll
          for (int d = 0; d < DD; ++d) {
            const f32x16_t hits = mfma32x32x16(v_frag(t, d, y), seen, zero16);
#pragma unroll
            for (int e = 0; e < 16; ++e) o[d][e] += hits[e] > 0.0f ? __builtin_nanf("") : 0.0f;
          }
        }
      }
    }
  }

  const int used = hi > lo ? (hi - lo + size - 1) / size : 1;
  const float sum = l + __shfl_xor(l, 32);
  if (row >= rows) return;
  const int64_t at = (sq.row0 + tok) * a.hq + head;
  if (NG > 1 || used == 1) {  // (two groups: there are blocks enough, no splits)
    const float f = sum != 0.0f ? 1.0f / sum : 0.0f;
#pragma unroll
    for (int d = 0; d < DD; ++d)
#pragma unroll
      for (int e = 0; e < 16; e += 4)
        store4<DT>(a.out, at * D + 32 * d + 2 * e + 4 * h, o[d][e] * f, o[d][e + 1] * f, o[d][e + 2] * f, o[d][e + 3] * f);
    if (h == 0 && a.lse) a.lse[at] = sum != 0.0f ? row_lse(m, sum) : -kInf;
  } else {
    const int64_t pr = at * a.splits + split;
#pragma unroll
    for (int d = 0; d < DD; ++d)
#pragma unroll
      for (int e = 0; e < 16; e += 4)
        *reinterpret_cast<f32x4_t*>(a.part_o + pr * D + 32 * d + 2 * e + 4 * h) = f32x4_t{o[d][e], o[d][e + 1], o[d][e + 2], o[d][e + 3]};
    if (h == 0) {
      a.part_ml[2 * pr] = m;
      a.part_ml[2 * pr + 1] = sum;
    }
  }
}

// Joins the splits of the many-rows kernel: one wave per row of the batch.
template <int DT, int D, int KT>
__global__ void __launch_bounds__(256) kv_attn_many_join_kernel(AttnArgs a, int64_t units) {
  constexpr int M = 128;
  const int64_t at = linear_block() * 4 + (threadIdx.x >> 6);
  if (at >= units) return;
  const int64_t t = at / a.hq;
  const int head = (int)(at - t * a.hq);
  const int b = find_sequence(a.seqs, t, [&](int i) { return (int64_t)a.cu[i]; });
  Seq sq;
  if (!seq_of(a, b, sq) || t < sq.row0 || t >= sq.row0 + sq.n || (int64_t)sq.n * a.group <= a.few_rows) return;
  const int r = (int)(t - sq.row0) * a.group + head % a.group;
  int lo, hi;
  many_keys<M>(a, sq, r / M * M, lo, hi);
  const int size = split_size(hi - lo, a.splits, KT);
  const int used = hi > lo ? (hi - lo + size - 1) / size : 1;
  if (used > 1) join_row<DT, D, 1>(a, used, at, [&](int x) { return at * a.splits + x; });
}

// ---- host -----------------------------------------------------------------------
int check(const char* fn, const pdm_kv_attention_desc* d, const pdm_kv_cache* c, const pdm_kv_batch* b) {
  auto bad = [&](const char* m) {
    set_error(std::string(fn) + ": " + m);
    return (int)PDM_ERR_INVALID;
  };
  if (!d || !c || !b) return bad("null descriptor");
  if (int e = check_cache(fn, c, b)) return e;
  if (d->dtype != PDM_F16 && d->dtype != PDM_BF16) return bad("dtype must be F16 or BF16");
  if (d->n_q_heads < 1 || d->n_q_heads % c->n_kv_heads) return bad("n_q_heads must be a multiple of n_kv_heads");
  if (d->n_q_heads / c->n_kv_heads > 1024) return bad("at most 1024 query heads per key head");
  if (d->window < 0) return bad("window must not be negative");
  if (!(d->scale - d->scale == 0.0f)) return bad("scale must be finite");
  if (d->max_q_len < 0) return bad("max_q_len must not be negative");
  if (b->tokens * d->n_q_heads >= (int64_t(1) << 31)) return bad("tokens * n_q_heads must be below 2^31");
  return PDM_OK;
}

// How a call is laid out, from its sizes alone (lengths are on the device).
struct Plan {
  int mt;                // tiles of 16 rows of the few-rows kernel
  bool few, many;        // which kernels may have work
  int splits, workers, row_stride;
  int64_t units, part_rows;
  int groups, many_splits;   // groups of 128 rows of the many-rows kernel
  int64_t items, many_part_rows;
};

Plan plan_of(const pdm_kv_attention_desc* d, const pdm_kv_cache* c, const pdm_kv_batch* b) {
  Plan p{};
  const int64_t group = d->n_q_heads / c->n_kv_heads;
  const int64_t max_q = d->max_q_len < b->tokens ? d->max_q_len : b->tokens;
  const int64_t rows = max_q * group;
  p.mt = c->head_dim == 256 || (group <= 16 && (rows <= 16 || rows > 32)) ? 1 : 2;
  p.splits = 1;
  if (b->num_seqs == 0) return p;  // padding alone: the few-rows kernel's blocks behind its units clear it
  p.few = group <= 16 * p.mt;
  p.many = rows > 16 * p.mt;
  const int64_t most = (int64_t)b->table_width * c->page_size;
  const int64_t pairs = (int64_t)b->num_seqs * c->n_kv_heads;
  const int64_t cap = (most + kFewStep - 1) / kFewStep;  // steps of a pair
  const int resident = 256 * (c->head_dim * p.mt <= 64 ? 4 : c->head_dim * p.mt <= 128 ? 3 : 2);
  // Dealt between the limits that it was made for and measured within (see few_deal): a sequence per thread, a pair for each CU
  // and more, up to eight times that, and partial results of 8 rows, two of each workgroup.  Outside them a batch gets equal
  // splits, or none from 1,024 pairs on, whatever its contexts; how much an uneven one loses by that has not been measured.
  p.workers = p.few && b->num_seqs > 1 && b->num_seqs <= kDealt && pairs >= 256 && pairs < 2048 && rows <= 8 && pairs * cap > resident
                  ? resident : 0;
  // else equal splits, as many as fill the CUs once: a second round of workgroups would only add joins
  int64_t splits = p.workers || pairs >= 1024 ? 1 : resident / pairs;
  splits = splits < cap ? splits : cap;
  p.splits = (int)(splits > 1 ? splits : 1);
  p.units = p.workers ? p.workers : pairs * p.splits;
  p.row_stride = (int)(rows < 16 * p.mt ? rows : 16 * p.mt);
  p.part_rows = !p.few ? 0 : p.workers ? 2 * p.workers * p.row_stride : p.splits > 1 ? p.units * p.row_stride : 0;
  if (p.many) {
    const int64_t all = b->tokens * group;
    // 256 rows a workgroup where they fill most of its blocks (256 rows a sequence on average) and there is one for each CU;
    // fewer rows would leave CUs idle.  Heads of 256 need the registers of two such waves for one.
    p.groups = c->head_dim < 256 && all >= 256 * (int64_t)b->num_seqs && all * c->n_kv_heads >= 256 * 256 ? 2 : 1;
    const int M = 128 * p.groups;
    p.items = all / M + b->num_seqs;
    // Blocks that are likely to have rows, where one sequence in five has many: too few for the CUs are split.  Behind 4,096
    // tokens, heads as above: 40 tokens of one of 64 sequences, single ones of the others 202 us unsplit, 146 split; 16 tokens of
    // 32 153 and 102.  (One in eight instead of five would split 10 tokens of 64 sequences, 38 -> 56 us behind 700 tokens.)
    const int64_t blocks = (all / M + 1 + b->num_seqs / 5) * c->n_kv_heads;
    int64_t sp = blocks < 256 && p.groups == 1 ? 512 / blocks : 1;
    const int64_t most_sp = (most + 511) / 512;
    sp = sp < most_sp ? sp : most_sp;
    p.many_splits = (int)(sp > 1 ? sp : 1);
    p.many_part_rows = p.many_splits > 1 ? b->tokens * d->n_q_heads * p.many_splits : 0;
  }
  return p;
}

int64_t round256(int64_t v) { return (v + 255) / 256 * 256; }

// The two kernels run one after the other, each with its join: they share the workspace.
int64_t part_rows_of(const Plan& p) { return p.part_rows > p.many_part_rows ? p.part_rows : p.many_part_rows; }
int64_t workspace_of(const Plan& p, int D) { return round256(part_rows_of(p) * D * 4) + round256(part_rows_of(p) * 8) + round256((int64_t)p.workers * 16); }

template <int DT, int D, int KT, int NG>
void launch_many(const AttnArgs& a, const Plan& p, hipStream_t st) {
  kv_attn_many_kernel<DT, D, KT, NG><<<linear_grid(p.items * a.hk * a.splits, (int64_t(1) << 23) / NG), 256 * NG, 0, st>>>(a, p.items);
  if constexpr (NG == 1)
    if (p.many_part_rows) {
      const int64_t rows = a.tokens * a.hq;
      kv_attn_many_join_kernel<DT, D, KT><<<linear_grid((rows + 3) / 4), 256, 0, st>>>(a, rows);
    }
}

template <int DT, int D>
void launch(AttnArgs& a, const Plan& p, hipStream_t st) {
  // `guards`: blocks that look for rows to clear and, where no unit looks at each sequence, at those, 256 of either
  const int64_t units = p.few ? p.units : 0, guards = ((units || a.tokens > a.seqs ? a.tokens : (int64_t)a.seqs) + 255) / 256;
  const dim3 grid = linear_grid(units + guards);
  if (p.mt == 1) kv_attn_few_kernel<DT, D, 1><<<grid, 256, 0, st>>>(a, units, guards);
  else if constexpr (D < 256) kv_attn_few_kernel<DT, D, 2><<<grid, 256, 0, st>>>(a, units, guards);  // more rows of 256 spill
  if (p.workers) {
    kv_attn_dealt_join_kernel<DT, D><<<(unsigned)p.workers, 256, 0, st>>>(a);
  } else if (p.part_rows) {
    const int64_t rows = (int64_t)a.seqs * a.hk * a.row_stride;
    if (rows < 4096) kv_attn_join_kernel<DT, D, 4><<<linear_grid(rows), 256, 0, st>>>(a, rows);
    else kv_attn_join_kernel<DT, D, 1><<<linear_grid((rows + 3) / 4), 256, 0, st>>>(a, rows);
  }
  if (!p.many) return;
  a.splits = p.many_splits;
  if constexpr (D == 256) launch_many<DT, D, 32, 1>(a, p, st);
  else if (p.groups == 2) launch_many<DT, D, 64, 2>(a, p, st);
  else launch_many<DT, D, 64, 1>(a, p, st);
}

template <int DT>
void launch_dt(AttnArgs& a, int D, const Plan& p, hipStream_t st) {
  if (D == 64) launch<DT, 64>(a, p, st);
  else if (D == 128) launch<DT, 128>(a, p, st);
  else launch<DT, 256>(a, p, st);
}

}  // namespace
}  // namespace pdm

using namespace pdm;

extern "C" int64_t pdm_kv_attention_workspace_size(const pdm_kv_attention_desc* d, const pdm_kv_cache* c,
                                                   const pdm_kv_batch* b) {
  clear_error();
  if (int e = check(__func__, d, c, b)) return e;
  return workspace_of(plan_of(d, c, b), c->head_dim);
}

extern "C" int pdm_kv_attention_fwd(const pdm_kv_attention_desc* d, const pdm_kv_cache* c, const pdm_kv_batch* b,
                                    const void* q, void* out, float* lse, void* workspace, int64_t workspace_bytes,
                                    int32_t* err_flag, pdm_stream_t stream) {
  clear_error();
  if (int e = check(__func__, d, c, b)) return e;
  if (b->tokens == 0) return PDM_OK;
  PDM_CHECK_ARG(q && out, "null q / out");
  PDM_CHECK_ARG((reinterpret_cast<uintptr_t>(out) & 15) == 0, "out must be 16-byte aligned");
  const Plan p = plan_of(d, c, b);
  const int64_t need = workspace_of(p, c->head_dim), o_bytes = round256(part_rows_of(p) * c->head_dim * 4);
  if (need && (!workspace || workspace_bytes < need)) {
    set_error(std::string(__func__) + ": workspace of " + std::to_string(need) + " bytes needed");
    return PDM_ERR_WORKSPACE;
  }
  PDM_CHECK_ARG((reinterpret_cast<uintptr_t>(workspace) & 255) == 0, "workspace must be 256-byte aligned");
  AttnArgs a{};
  a.q = q, a.out = out, a.lse = lse;
  a.k_codes = c->k_codes, a.v_codes = c->v_codes, a.k_scale = c->k_scale, a.v_scale = c->v_scale;
  a.cu = b->cu_seqlens, a.table = b->page_table, a.lens = b->seq_lens, a.err = err_flag;
  a.part_o = static_cast<float*>(workspace);
  a.part_ml = reinterpret_cast<float*>(static_cast<char*>(workspace) + o_bytes);
  a.joins = reinterpret_cast<int32_t*>(static_cast<char*>(workspace) + o_bytes + round256(part_rows_of(p) * 8));
  a.tokens = b->tokens, a.table_stride = b->table_stride, a.num_pages = c->num_pages;
  a.stride_t = d->q_stride_t, a.stride_h = d->q_stride_h;
  a.seqs = b->num_seqs, a.hq = d->n_q_heads, a.hk = c->n_kv_heads, a.group = d->n_q_heads / c->n_kv_heads;
  a.page_log2 = log2_of(c->page_size), a.table_width = b->table_width;
  a.max_q = d->max_q_len;
  a.causal = d->causal != 0, a.window = d->window;
  a.splits = p.splits, a.workers = p.workers, a.row_stride = p.row_stride, a.few_rows = p.few ? 16 * p.mt : 0;
  a.vec = (reinterpret_cast<uintptr_t>(q) & 15) == 0 && d->q_stride_t % 8 == 0 && d->q_stride_h % 8 == 0;
  a.scale2 = d->scale * 1.44269504088896341f;
  if (d->dtype == PDM_BF16) launch_dt<PDM_BF16>(a, c->head_dim, p, stream);
  else launch_dt<PDM_F16>(a, c->head_dim, p, stream);
  PDM_CHECK_LAUNCH();
  return PDM_OK;
}
