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
// holds exactly.  Weights are rounded to bf16 (half a step is 2^-8 of a weight, against 2^-4 of an 8-bit value);
// the running sum takes them before that.
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
  int64_t tokens, table_stride, num_pages, stride_t, stride_h;
  int32_t seqs, hq, hk, group, page_log2, table_width, max_q, causal, window;
  int32_t splits;            // of the keys of a (sequence, key head)
  int32_t row_stride;        // rows of a partial result
  int32_t few_rows;          // sequences of at most so many rows are kv_attn_few_kernel's
  int32_t vec;               // q takes 16-byte loads
  float scale2;              // scale * log2(e)
};

constexpr float kInf = __builtin_inff();
constexpr float kLn2 = 0.69314718055994531f;

// What a sequence's rows see.
struct Seq {
  int64_t row0;   // its first row of the batch
  int n, len;     // new tokens, length
  int lo, hi;     // keys that any of its rows may see, lo a multiple of 32
};

__device__ __forceinline__ bool seq_fits(const AttnArgs& a, int64_t c0, int64_t c1, int64_t len) {
  return c0 >= 0 && c1 <= a.tokens && c1 - c0 <= a.max_q && c1 - c0 <= len;
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
  const int64_t most = (int64_t)a.table_width << a.page_log2;
  s.hi = (int)(len < most ? len : most);
  if (len > most && a.err) *a.err = 1;
  const int64_t first = len - s.n - a.window + 1;
  s.lo = a.window > 0 && first > 0 ? (int)first & ~31 : 0;
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

// NaN codes of a dword: bit 7 of each byte that holds one.
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }

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
  __syncthreads();
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
// has the next tile's loads (8 KB at D = 128) in flight while it works on one.
constexpr int kFewKeys = 32, kFewWaves = 4;

template <int D>
struct FewTile {
  static constexpr int KC = D / 64;       // 16-byte pieces of a key row per lane
  static constexpr int VW = D / 64;       // dwords of a value row per lane
  u32x4_t k[2][KC];                       // 16 keys each
  uint32_t v[2][4][VW];                   // rows 4 g + i of the 16 keys
  float ks[2], vs[2];
  bool ok[2];
};

template <int DT, int D, int MT>
__global__ void __launch_bounds__(256) kv_attn_few_kernel(AttnArgs a, int64_t units, int64_t guards) {
  constexpr int KK = D / 32;              // steps of the first product
  constexpr int DD = D / 16;              // tiles of the second: O^T row m of tile dd is element DD m + dd
  __shared__ float red[kFewWaves][16][D + 4];
  __shared__ float ml[kFewWaves][2][16 * MT];
  const int64_t unit = linear_block();
  if (unit >= units) {
    if (unit < units + guards) clear_rows<D>(a, (unit - units) * 256);
    return;
  }
  const int split = (int)(unit % a.splits);
  const int64_t bh = unit / a.splits;
  const int kh = (int)(bh % a.hk), b = (int)(bh / a.hk);
  Seq sq;
  if (!seq_of(a, b, sq)) return;
  const int rows = sq.n * a.group;
  if (rows > a.few_rows) return;
  const int size = split_size(sq.hi - sq.lo, a.splits, kFewKeys * kFewWaves);
  const int begin = sq.lo + split * size;
  if (split > 0 && begin >= sq.hi) return;
  const int end = begin + size < sq.hi ? begin + size : sq.hi;

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4;

  // this lane's rows: queries, and the keys that they see
  u32x4_t q[MT][KK];
  int row_lo[MT], row_hi[MT];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    const int r = mt * 16 + c;
    const int i = r / a.group, h = kh * a.group + (r - i * a.group);
    row_lo[mt] = 0x7fffffff, row_hi[mt] = 0;
    if (r < rows) {
      const int p = sq.len - sq.n + i;
      row_hi[mt] = a.causal && p + 1 < sq.hi ? p + 1 : sq.hi;
      row_lo[mt] = a.window > 0 && p - a.window + 1 > 0 ? p - a.window + 1 : 0;
      const uint16_t* x = static_cast<const uint16_t*>(a.q) + (sq.row0 + i) * a.stride_t + h * a.stride_h;
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) {
        const uint16_t* p8 = x + 64 * (kk >> 1) + 16 * g + 8 * (kk & 1);
        if (a.vec) {
          q[mt][kk] = *reinterpret_cast<const u32x4_t*>(p8);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) q[mt][kk][e] = uint32_t(p8[2 * e]) | uint32_t(p8[2 * e + 1]) << 16;
        }
      }
    } else {
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) q[mt][kk] = u32x4_t{0, 0, 0, 0};
    }
  }
  // keys that every row sees (rows that are not there do not count)
  int all_lo = 0, all_hi = sq.hi;
  {
    const int p0 = sq.len - sq.n, p1 = sq.len - 1;
    if (a.causal && p0 + 1 < all_hi) all_hi = p0 + 1;
    if (a.window > 0 && p1 - a.window + 1 > 0) all_lo = p1 - a.window + 1;
  }

  float m[MT], l[MT];
  f32x4_t o[MT][DD];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    m[mt] = -kInf, l[mt] = 0.0f;
#pragma unroll
    for (int d = 0; d < DD; ++d) o[mt][d] = f32x4_t{0, 0, 0, 0};
  }

  const int32_t* table = a.table + (int64_t)b * a.table_stride;
  const int tiles = (end - begin + kFewKeys - 1) / kFewKeys;
  const int mine = tiles > wave ? (tiles - wave + kFewWaves - 1) / kFewWaves : 0;

  // lane i of a batch of 32 tiles: page and scales of the 16 keys i % 2 of tile i / 2
  int ids = -1;
  float kss = 0.0f, vss = 0.0f;
  auto look_up = [&](int first) {
    const int key = begin + (wave + kFewWaves * (first + (lane >> 1))) * kFewKeys + (lane & 1) * 16;
    ids = -1;
    if (key < end) {
      const int id = table[key >> a.page_log2];
      if (id >= 0 && id < a.num_pages) {
        ids = id;
        const int64_t entry = (int64_t)id * a.hk + kh;
        kss = a.k_scale[entry];
        vss = a.v_scale[entry];
      } else if (a.err) {
        *a.err = 1;
      }
    }
  };
  const uint32_t k_off = (uint32_t)(c * D + 16 * g);
  const uint32_t v_off = (uint32_t)(4 * g * D + (D / 16) * c);
  auto load = [&](FewTile<D>& t, int i) {
    if ((i & 31) == 0) look_up(i);
    const int key = begin + (wave + kFewWaves * i) * kFewKeys;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int x = (i & 31) * 2 + s;
      const int id = __builtin_amdgcn_readlane(ids, x);
      t.ok[s] = id >= 0;
      t.ks[s] = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, kss), x));
      t.vs[s] = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, vss), x));
      if (!t.ok[s]) {
#pragma unroll
        for (int e = 0; e < FewTile<D>::KC; ++e) t.k[s][e] = u32x4_t{0, 0, 0, 0};
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int e = 0; e < FewTile<D>::VW; ++e) t.v[s][r][e] = 0;
        continue;
      }
      const int64_t row = (((int64_t)id * a.hk + kh) << a.page_log2) + ((key + 16 * s) & ((1 << a.page_log2) - 1));
      const uint8_t* kp = a.k_codes + row * D + k_off;
      const uint8_t* vp = a.v_codes + row * D + v_off;
#pragma unroll
      for (int e = 0; e < FewTile<D>::KC; ++e) t.k[s][e] = *reinterpret_cast<const u32x4_t*>(kp + 64 * e);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        if constexpr (D == 64) {
          t.v[s][r][0] = *reinterpret_cast<const uint32_t*>(vp + r * D);
        } else if constexpr (D == 128) {
          const u32x2_t w = *reinterpret_cast<const u32x2_t*>(vp + r * D);
          t.v[s][r][0] = w[0], t.v[s][r][1] = w[1];
        } else {
          const u32x4_t w = *reinterpret_cast<const u32x4_t*>(vp + r * D);
#pragma unroll
          for (int e = 0; e < 4; ++e) t.v[s][r][e] = w[e];
        }
      }
    }
  };

  auto work = [&](FewTile<D>& t, int i) {
    const int key = begin + (wave + kFewWaves * i) * kFewKeys;
    f32x4_t s[MT][2];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) s[mt][x] = f32x4_t{0, 0, 0, 0};
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) {
        const uint32_t w0 = t.k[x][kk >> 1][2 * (kk & 1)], w1 = t.k[x][kk >> 1][2 * (kk & 1) + 1];
        const u32x4_t kf = {code_pair<DT>(w0, false), code_pair<DT>(w0, true), code_pair<DT>(w1, false), code_pair<DT>(w1, true)};
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) s[mt][x] = mfma16<DT>(kf, q[mt][kk], s[mt][x]);
      }
    }
    const bool whole = t.ok[0] && t.ok[1] && key >= all_lo && key + kFewKeys <= all_hi;
    u32x4_t p[MT], seen[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = s[mt][e >> 2][e & 3] * (a.scale2 * t.ks[e >> 2]);
      uint32_t sees = 0xffu;
      if (!whole) {
        sees = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int j = key + 16 * (e >> 2) + 4 * g + (e & 3);
          const bool on = t.ok[e >> 2] && j >= row_lo[mt] && j < row_hi[mt];
          v[e] = on ? v[e] : -kInf;
          sees |= on ? 1u << e : 0u;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
          seen[mt][e] = ((sees >> (2 * e)) & 1u ? 0x3f80u : 0u) | ((sees >> (2 * e + 1)) & 1u ? 0x3f800000u : 0u);
      }
      float top = v[0];
#pragma unroll
      for (int e = 1; e < 8; ++e) top = fmaxf(top, v[e]);
      // the maximum moves only where a weight would pass 2^8: sums and products lose nothing by that
      if (__any(top > m[mt] + 8.0f)) {
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
        const float now = top > m[mt] + 8.0f ? top : m[mt];  // by row: other rows change nothing
        const float f = now == -kInf ? 1.0f : __builtin_amdgcn_exp2f(m[mt] - now);
        m[mt] = now;
        l[mt] *= f;
#pragma unroll
        for (int d = 0; d < DD; ++d) o[mt][d] *= f;
      }
      const float base = m[mt] == -kInf ? 0.0f : m[mt];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = __builtin_amdgcn_exp2f(v[e] - base);
      l[mt] += ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
      p[mt] = u32x4_t{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7])};
    }
    // a NaN value must not reach rows that do not see it (0 * NaN): in a tile that some row sees in part, NaN codes are
    // taken out and counted by a product of their own
    bool odd = false;
    if (!whole) {
      uint32_t any = 0;
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int e = 0; e < FewTile<D>::VW; ++e) any |= nan_bytes(t.v[x][r][e]);
      odd = __any(any != 0);
    }
#pragma unroll
    for (int h = 0; h < FewTile<D>::VW; ++h) {
      // 4 x 4 bytes (keys x elements) of each 16 keys, turned to pairs of keys
      uint32_t w01[2][2], w23[2][2];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        w01[x][0] = __builtin_amdgcn_perm(t.v[x][1][h], t.v[x][0][h], 0x05010400u);
        w01[x][1] = __builtin_amdgcn_perm(t.v[x][1][h], t.v[x][0][h], 0x07030602u);
        w23[x][0] = __builtin_amdgcn_perm(t.v[x][3][h], t.v[x][2][h], 0x05010400u);
        w23[x][1] = __builtin_amdgcn_perm(t.v[x][3][h], t.v[x][2][h], 0x07030602u);
      }
      if (odd) {
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          u32x4_t ones;
          const bool hi = x & 1;
          const uint32_t src[4] = {w01[0][x >> 1], w23[0][x >> 1], w01[1][x >> 1], w23[1][x >> 1]};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t nb = nan_bytes(src[e]) >> (hi ? 16 : 0);
            ones[e] = (nb & 0x80u ? 0x3f80u : 0u) | (nb & 0x8000u ? 0x3f800000u : 0u);
          }
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            const f32x4_t hits = mfma16x16x32(ones, seen[mt], f32x4_t{0, 0, 0, 0});
#pragma unroll
            for (int e = 0; e < 4; ++e) o[mt][4 * h + x][e] += hits[e] > 0.0f ? __builtin_nanf("") : 0.0f;
          }
        }
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const uint32_t n0 = nan_bytes(w01[x][e]), n1 = nan_bytes(w23[x][e]);
            w01[x][e] &= ~((n0 >> 7) * 0xffu);
            w23[x][e] &= ~((n1 >> 7) * 0xffu);
          }
      }
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int hf = x >> 1;
        const u32x4_t vf = x & 1 ? u32x4_t{value_pair_hi(w01[0][hf], t.vs[0]), value_pair_hi(w23[0][hf], t.vs[0]),
                                           value_pair_hi(w01[1][hf], t.vs[1]), value_pair_hi(w23[1][hf], t.vs[1])}
                                 : u32x4_t{value_pair_lo(w01[0][hf], t.vs[0]), value_pair_lo(w23[0][hf], t.vs[0]),
                                           value_pair_lo(w01[1][hf], t.vs[1]), value_pair_lo(w23[1][hf], t.vs[1])};
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) o[mt][4 * h + x] = mfma16x16x32(vf, p[mt], o[mt][4 * h + x]);
      }
    }
  };

  if constexpr (D * MT > 256) {  // the registers hold one tile
    for (int i = 0; i < mine; ++i) {
      FewTile<D> t0;
      load(t0, i);
      work(t0, i);
    }
  } else if (mine > 0) {
    FewTile<D> t0, t1;
    load(t0, 0);
    for (int i = 0; i < mine; i += 2) {
      if (i + 1 < mine) load(t1, i + 1);
      work(t0, i);
      if (i + 1 < mine) {
        if (i + 2 < mine) load(t0, i + 2);
        work(t1, i + 1);
      }
    }
  }

  // join the waves: the sums of a row are spread over its four lanes
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    l[mt] += __shfl_xor(l[mt], 16);
    l[mt] += __shfl_xor(l[mt], 32);
    if (g == 0) {
      ml[wave][0][mt * 16 + c] = m[mt];
      ml[wave][1][mt * 16 + c] = l[mt];
    }
  }
  __syncthreads();
  const int used = sq.hi > sq.lo ? (sq.hi - sq.lo + size - 1) / size : 1;
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    const int r = mt * 16 + c;
    float top = ml[0][0][r];
#pragma unroll
    for (int w = 1; w < kFewWaves; ++w) top = fmaxf(top, ml[w][0][r]);
    const float f = m[mt] == -kInf ? (l[mt] != l[mt] ? 1.0f : 0.0f) : __builtin_amdgcn_exp2f(m[mt] - top);
    if (mt) __syncthreads();
    if (r < rows) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int d = 0; d < DD; d += 4)
          *reinterpret_cast<f32x4_t*>(&red[wave][c][DD * (4 * g + e) + d]) =
              f32x4_t{o[mt][d][e] * f, o[mt][d + 1][e] * f, o[mt][d + 2][e] * f, o[mt][d + 3][e] * f};
    }
    __syncthreads();
    for (int x = threadIdx.x; x < 16 * D; x += 256) {
      const int rr = x / D, d = x - rr * D, row = mt * 16 + rr;
      if (row >= rows) break;
      float top_r = ml[0][0][row];
#pragma unroll
      for (int w = 1; w < kFewWaves; ++w) top_r = fmaxf(top_r, ml[w][0][row]);
      float sum = 0.0f, acc = 0.0f;
#pragma unroll
      for (int w = 0; w < kFewWaves; ++w) {
        const float lw = ml[w][1][row];
        sum += lw * (ml[w][0][row] == -kInf ? 1.0f : __builtin_amdgcn_exp2f(ml[w][0][row] - top_r));
        acc += red[w][rr][d];
      }
      if (used == 1) {
        const int i = row / a.group, h = kh * a.group + (row - i * a.group);
        const int64_t at = (sq.row0 + i) * a.hq + h;
        store_out(a, DT, at * D + d, sum != 0.0f ? acc / sum : 0.0f);
        if (d == 0 && a.lse) a.lse[at] = sum != 0.0f ? (top_r + __builtin_amdgcn_logf(sum)) * kLn2 : -kInf;
      } else {
        const int64_t at = unit * a.row_stride + row;
        a.part_o[at * D + d] = acc;
        if (d == 0) {
          a.part_ml[2 * at] = top_r;
          a.part_ml[2 * at + 1] = sum;
        }
      }
    }
  }
}

// Joins the `used` partial results of one row, `step` rows apart from `first`; one wave.
template <int DT, int D>
__device__ __forceinline__ void join_row(const AttnArgs& a, int64_t first, int64_t step, int used, int64_t at) {
  constexpr int E = D / 64;
  const int lane = threadIdx.x & 63;
  float top = -kInf;
  for (int s = lane; s < used; s += 64) top = fmaxf(top, a.part_ml[2 * (first + s * step)]);
  top = group_max(top, 64);
  float sum = 0.0f, acc[E];
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = 0.0f;
#pragma unroll 4
  for (int s = 0; s < used; ++s) {
    const int64_t pr = first + s * step;
    const float m = a.part_ml[2 * pr], l = a.part_ml[2 * pr + 1];
    const float f = m == -kInf ? (l != l ? 1.0f : 0.0f) : __builtin_amdgcn_exp2f(m - top);
    sum += l * f;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] += a.part_o[pr * D + lane * E + e] * f;
  }
#pragma unroll
  for (int e = 0; e < E; ++e) store_out(a, DT, at * D + lane * E + e, sum != 0.0f ? acc[e] / sum : 0.0f);
  if (lane == 0 && a.lse) a.lse[at] = sum != 0.0f ? (top + __builtin_amdgcn_logf(sum)) * kLn2 : -kInf;
}

// Joins the splits of the few-rows kernel: one wave per row.
template <int DT, int D>
__global__ void __launch_bounds__(256) kv_attn_join_kernel(AttnArgs a, int64_t units) {
  const int64_t x = linear_block() * 4 + (threadIdx.x >> 6);
  if (x >= units) return;
  const int row = (int)(x % a.row_stride);
  const int64_t bh = x / a.row_stride;
  const int kh = (int)(bh % a.hk), b = (int)(bh / a.hk);
  Seq sq;
  if (!seq_of(a, b, sq)) return;
  const int64_t rows = (int64_t)sq.n * a.group;
  if (rows > a.few_rows || row >= rows) return;
  const int size = split_size(sq.hi - sq.lo, a.splits, kFewKeys * kFewWaves);
  const int used = sq.hi > sq.lo ? (sq.hi - sq.lo + size - 1) / size : 1;
  if (used == 1) return;
  const int i = row / a.group, h = kh * a.group + (row - i * a.group);
  join_row<DT, D>(a, bh * a.splits * a.row_stride + row, a.row_stride, used, (sq.row0 + i) * a.hq + h);
}

// ---- many rows ---------------------------------------------------------------------
// 128 rows of a (sequence, key head) against its keys, four waves of 32 rows.  Tiles of KT keys are converted once on
// their way into LDS: K as rows, two tiles ahead of the values' use, V transposed, one tile ahead, its keys in the order in
// which the first product leaves P.  The waves meet at one barrier per tile.  A wave computes the scores of tile t + 1
// beside the exponentials of tile t, and a second workgroup shares the CU: the matrix unit has work while the VALU does
// a softmax.
constexpr int kManyRows = 128;

template <int D, int KT>
struct ManyShared {
  static constexpr int KS = 2 * D + 16;    // bytes of a K row: 16 rows of a fragment read fall into different banks
  static constexpr int VS = 2 * KT + 16;   // bytes of a V^T row
  alignas(16) char k[2][KT * KS];
  alignas(16) char v[2][D * VS];
  float sc[4][KT / 16];                    // scale2 * scale of 16 keys; NaN where their page does not exist
  int odd[4];                              // a wave's share of V held NaN
};

// Block `item` of the list of (sequence, 128 rows): sequence b's span begins at cu[b] * group / 128 + b.
__device__ __forceinline__ bool many_block(const AttnArgs& a, int64_t item, Seq& sq, int& b, int& r0) {
  b = find_sequence(a.seqs, item, [&](int i) { return (int64_t)a.cu[i] * a.group / kManyRows + i; });
  const int64_t j = item - ((int64_t)a.cu[b] * a.group / kManyRows + b);
  if (j < 0 || !seq_of(a, b, sq)) return false;
  const int64_t rows = (int64_t)sq.n * a.group;
  if (rows <= a.few_rows || j * kManyRows >= rows) return false;
  r0 = (int)(j * kManyRows);
  return true;
}

// The keys that rows r0 .. r0 + 127 may see: [lo, hi), lo a multiple of 32.
__device__ __forceinline__ void many_keys(const AttnArgs& a, const Seq& sq, int r0, int& lo, int& hi) {
  const int rows = sq.n * a.group;
  const int i0 = r0 / a.group, i1 = ((r0 + kManyRows < rows ? r0 + kManyRows : rows) - 1) / a.group;
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

template <int DT, int D, int KT>
__global__ void __launch_bounds__(256, D == 256 ? 1 : 2) kv_attn_many_kernel(AttnArgs a, int64_t items) {
  constexpr int KK = D / 16, DD = D / 32, XX = KT / 32;
  constexpr int KP = KT * D / 16 / 256;    // 16-byte pieces of a K tile per thread
  constexpr int VD = D == 64 ? 4 : 8;      // elements of a thread's 4 keys of V
  constexpr int KS = ManyShared<D, KT>::KS, VS = ManyShared<D, KT>::VS;
  __shared__ ManyShared<D, KT> sh;

  const int64_t unit = linear_block();
  const int split = (int)(unit % a.splits);
  const int64_t ih = unit / a.splits;
  const int kh = (int)(ih % a.hk);
  const int64_t item = items - 1 - ih / a.hk;  // later rows see more keys: they begin first
  if (item < 0) return;
  Seq sq;
  int b, r0;
  if (!many_block(a, item, sq, b, r0)) return;
  int lo, hi;
  many_keys(a, sq, r0, lo, hi);
  const int size = split_size(hi - lo, a.splits, KT);
  const int begin = lo + split * size;
  if (split > 0 && begin >= hi) return;
  const int end = begin + size < hi ? begin + size : hi;
  const int rows = sq.n * a.group;
  const int tiles = end > begin ? (end - begin + KT - 1) / KT : 0;

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 31, h = lane >> 5;

  // this lane's row: its query, and the keys that it sees
  u32x4_t q[KK];
  int row_lo = 0x7fffffff, row_hi = 0;
  const int row = r0 + wave * 32 + c;
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
  // keys that every row of this wave sees
  int all_lo = 0, all_hi = sq.hi;
  {
    const int w0 = r0 + wave * 32;
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
  int ids = -1;                            // lane i: page and scales of keys 16 i .. of the batch
  float kss = 0.0f, vss = 0.0f;
  u32x4_t kr[KP];
  uint32_t vr[4][VD / 4];
  int v_id = -1;                           // of the V tile that is loaded next
  float v_sc = 0.0f, v_scale = 0.0f, sc_reg = 0.0f;
  const int kc = (tid % (D / 16)) * 16, kr0 = tid / (D / 16);       // piece and row of K, 4096 / D rows a pass
  const int vm = D == 256 ? wave * 8 + (lane & 7) : (wave & 1) * 8 + (lane & 7);
  const int va = D == 256 ? lane >> 3 : (wave >> 1) * 8 + (lane >> 3);   // four keys of V
  auto load_k = [&](int t) {
    const int key0 = begin + t * KT;
    if (t % PER == 0) {
      const int key = key0 + 16 * lane;
      ids = -1, kss = __builtin_nanf(""), vss = 0.0f;
      if (key < end) {
        const int id = table[key >> a.page_log2];
        if (id >= 0 && id < a.num_pages) {
          ids = id;
          const int64_t entry = (int64_t)id * a.hk + kh;
          kss = a.k_scale[entry] * a.scale2;
          vss = a.v_scale[entry];
        } else if (a.err) {
          *a.err = 1;
        }
      }
    }
    const int g0 = (t % PER) * (KT / 16);
#pragma unroll
    for (int p = 0; p < KP; ++p) {
      const int r = kr0 + p * (4096 / D);
      const int grp = __builtin_amdgcn_readfirstlane(r >> 4);
      const int id = __builtin_amdgcn_readlane(ids, g0 + grp);
      kr[p] = u32x4_t{0, 0, 0, 0};
      if (id >= 0) {
        const int64_t at = (((int64_t)id * a.hk + kh) << a.page_log2) + ((key0 + 16 * grp) & mask);
        kr[p] = *reinterpret_cast<const u32x4_t*>(a.k_codes + at * D + (r & 15) * D + kc);
      }
    }
    v_id = __shfl(ids, g0 + (va >> 2));
    v_sc = __shfl(vss, g0 + (va >> 2));
    sc_reg = __shfl(kss, g0 + (lane & (KT / 16 - 1)));
  };
  auto load_v = [&](int t) {  // with the page that load_k(t) found
    v_scale = v_sc;
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int e = 0; e < VD / 4; ++e) vr[r][e] = 0;
    if (v_id >= 0) {
      const int64_t at = (((int64_t)v_id * a.hk + kh) << a.page_log2) + ((begin + t * KT + 16 * (va >> 2)) & mask) + (va & 3) * 4;
      const uint8_t* p = a.v_codes + at * D + vm * VD;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        if constexpr (VD == 4) {
          vr[r][0] = *reinterpret_cast<const uint32_t*>(p + r * D);
        } else {
          const u32x2_t w = *reinterpret_cast<const u32x2_t*>(p + r * D);
          vr[r][0] = w[0], vr[r][1] = w[1];
        }
      }
    }
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
    if (wave == 0 && lane < KT / 16) sh.sc[t & 3][lane] = sc_reg;
  };
  // V^T of tile t; NaN codes become zeros here (0 * NaN would reach rows that do not see the key) and are remembered, or,
  // in MARK, ones where everything else becomes zero.
  bool odd = false;
  auto stage_v = [&](int t, auto mark) {
    // keys 4 va .. + 3: block va % 4 of their 16; blocks 0, 2 belong to lanes h = 0 of the product, 1, 3 to h = 1
    const int x = va & 3;
    char* vb = sh.v[t & 1] + 2 * (16 * (va >> 2) + 8 * (x & 1) + 4 * (x >> 1));
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
          for (int r = 0; r < 4; ++r) vr[r][e] &= ~((nan_bytes(vr[r][e]) >> 7) * 0xffu);
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
        *reinterpret_cast<u32x2_t*>(vb + (vm * VD + 4 * e + d) * VS) = w;
      }
    }
  };

  // ---- products ----
  float m = -kInf, l = 0.0f;
  f32x16_t o[DD], s[XX], n[XX];
  constexpr f32x16_t zero16 = {0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
  for (int d = 0; d < DD; ++d) o[d] = zero16;
  const uint32_t k_at = c * KS + 16 * h, v_at = c * VS + 16 * h;
  auto scores = [&](int t) {
    const char* kb = sh.k[t & 1] + k_at;
#pragma unroll
    for (int x = 0; x < XX; ++x) {
      n[x] = zero16;
#pragma unroll
      for (int kk = 0; kk < KK; ++kk)
        n[x] = mfma32<DT>(*reinterpret_cast<const u32x4_t*>(kb + x * 32 * KS + 32 * kk), q[kk], n[x]);
    }
  };
  // s = the new scores in units of log2, hidden ones at -inf; the running maximum
  auto settle = [&](int t) {
    const int key = begin + t * KT;
    float sc[2 * XX];
    bool ok = true;
#pragma unroll
    for (int x = 0; x < 2 * XX; ++x) {
      sc[x] = __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, sh.sc[t & 3][x])));
      ok = ok && sc[x] == sc[x];
    }
#pragma unroll
    for (int x = 0; x < XX; ++x)
#pragma unroll
      for (int e = 0; e < 16; ++e) s[x][e] = n[x][e] * sc[2 * x + (e >> 3)];
    if (!(ok && key >= all_lo && key + KT <= all_hi)) {
#pragma unroll
      for (int x = 0; x < XX; ++x)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int j = key + 32 * x + 8 * (e >> 2) + 4 * h + (e & 3);
          const bool on = sc[2 * x + (e >> 3)] == sc[2 * x + (e >> 3)] && j >= row_lo && j < row_hi;
          s[x][e] = on ? s[x][e] : -kInf;
        }
    }
    float top = s[0][0];
#pragma unroll
    for (int x = 0; x < XX; ++x)
#pragma unroll
      for (int e = 0; e < 16; ++e) top = fmaxf(top, s[x][e]);
    // the maximum moves only where a weight would pass 2^8: sums and products lose nothing by that
    if (__any(top > m + 8.0f)) {
      top = fmaxf(top, __shfl_xor(top, 32));
      const float now = top > m + 8.0f ? top : m;  // by row: other rows change nothing
      const float f = now == -kInf ? 1.0f : __builtin_amdgcn_exp2f(m - now);
      m = now;
      l *= f;
#pragma unroll
      for (int d = 0; d < DD; ++d) o[d] *= f;
    }
  };
  u32x4_t p[2 * XX];
  auto weights = [&]() {
    const float base = m == -kInf ? 0.0f : m;
#pragma unroll
    for (int x = 0; x < XX; ++x) {
      float v[16];
#pragma unroll
      for (int e = 0; e < 16; ++e) v[e] = __builtin_amdgcn_exp2f(s[x][e] - base);
#pragma unroll
      for (int e = 0; e < 16; e += 4) l += (v[e] + v[e + 1]) + (v[e + 2] + v[e + 3]);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        p[2 * x][e] = pack_bf16x2(v[2 * e], v[2 * e + 1]);
        p[2 * x + 1][e] = pack_bf16x2(v[8 + 2 * e], v[8 + 2 * e + 1]);
      }
    }
  };
  auto values = [&](int t) {
    const char* vb = sh.v[t & 1] + v_at;
#pragma unroll
    for (int y = 0; y < 2 * XX; ++y)
#pragma unroll
      for (int d = 0; d < DD; ++d)
        o[d] = mfma32x32x16(*reinterpret_cast<const u32x4_t*>(vb + d * 32 * VS + 32 * y), p[y], o[d]);
  };
  if (tiles > 0) {
    const std::false_type plain;
    load_k(0);
    load_v(0);
    stage_k(0);
    stage_v(0, plain);
    if (tiles > 1) {
      load_k(1);
      load_v(1);
      stage_k(1);
    }
    if (tiles > 2) load_k(2);
    __syncthreads();
    scores(0);
    settle(0);
#pragma unroll 1
    for (int t = 0; t + 1 < tiles; ++t) {
      __syncthreads();
      stage_v(t + 1, plain);
      if (t + 2 < tiles) {
        load_v(t + 2);
        stage_k(t + 2);
        if (t + 3 < tiles) load_k(t + 3);
      }
      scores(t + 1);
      weights();
      values(t);
      settle(t + 1);
    }
    __syncthreads();
    weights();
    values(tiles - 1);

    // NaN among the values of any wave's share: once more over the tiles, with ones for NaN and for keys that are seen
    if (lane == 0) sh.odd[wave] = odd;
    __syncthreads();
    if (sh.odd[0] | sh.odd[1] | sh.odd[2] | sh.odd[3]) {
#pragma unroll 1
      for (int t = 0; t < tiles; ++t) {
        load_k(t);
        load_v(t);
        __syncthreads();  // the tile before is done with
        stage_v(t, std::true_type());
        if (wave == 0 && lane < KT / 16) sh.sc[t & 3][lane] = sc_reg;
        __syncthreads();
#pragma unroll 1
        for (int y = 0; y < 2 * XX; ++y) {
          u32x4_t seen;
          const bool ok = sh.sc[t & 3][y] == sh.sc[t & 3][y];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int j = begin + t * KT + 16 * y + 8 * (e >> 1) + 4 * h + 2 * (e & 1);
            seen[e] = (ok && j >= row_lo && j < row_hi ? 0x3f80u : 0u) | (ok && j + 1 >= row_lo && j + 1 < row_hi ? 0x3f800000u : 0u);
          }
#pragma unroll
          for (int d = 0; d < DD; ++d) {
            const f32x16_t hits = mfma32x32x16(*reinterpret_cast<const u32x4_t*>(sh.v[t & 1] + v_at + d * 32 * VS + 32 * y), seen, zero16);
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
  if (used == 1) {
    const float f = sum != 0.0f ? 1.0f / sum : 0.0f;
#pragma unroll
    for (int d = 0; d < DD; ++d)
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        const float w[4] = {o[d][e] * f, o[d][e + 1] * f, o[d][e + 2] * f, o[d][e + 3] * f};
        u32x2_t y;
        if constexpr (DT == PDM_BF16) {
          y = u32x2_t{pack_bf16x2(w[0], w[1]), pack_bf16x2(w[2], w[3])};
        } else {
          y = u32x2_t{f32_to_f16_bits(w[0]) | f32_to_f16_bits(w[1]) << 16, f32_to_f16_bits(w[2]) | f32_to_f16_bits(w[3]) << 16};
        }
        *reinterpret_cast<u32x2_t*>(static_cast<uint16_t*>(a.out) + at * D + 32 * d + 2 * e + 4 * h) = y;
      }
    if (h == 0 && a.lse) a.lse[at] = sum != 0.0f ? (m + __builtin_amdgcn_logf(sum)) * kLn2 : -kInf;
  } else {
    const int64_t pr = ((item * a.hk + kh) * a.splits + split) * kManyRows + wave * 32 + c;
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

// Joins the splits of the many-rows kernel: one wave per row.
template <int DT, int D, int KT>
__global__ void __launch_bounds__(256) kv_attn_many_join_kernel(AttnArgs a, int64_t items) {
  const int64_t x = linear_block() * 4 + (threadIdx.x >> 6);
  const int in = (int)(x % kManyRows);
  const int64_t ih = x / kManyRows;
  const int kh = (int)(ih % a.hk);
  const int64_t item = ih / a.hk;
  if (item >= items) return;
  Seq sq;
  int b, r0, lo, hi;
  if (!many_block(a, item, sq, b, r0)) return;
  const int r = r0 + in;
  if (r >= sq.n * a.group) return;
  many_keys(a, sq, r0, lo, hi);
  const int size = split_size(hi - lo, a.splits, KT);
  const int used = hi > lo ? (hi - lo + size - 1) / size : 1;
  if (used == 1) return;
  const int i = r / a.group, h = kh * a.group + (r - i * a.group);
  join_row<DT, D>(a, ih * a.splits * kManyRows + in, kManyRows, used, (sq.row0 + i) * a.hq + h);
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
  int splits, row_stride;
  int64_t part_rows;
  int many_splits;
  int64_t items, many_part_rows;
};

Plan plan_of(const pdm_kv_attention_desc* d, const pdm_kv_cache* c, const pdm_kv_batch* b) {
  Plan p{};
  const int64_t group = d->n_q_heads / c->n_kv_heads;
  const int64_t max_q = d->max_q_len < b->tokens ? d->max_q_len : b->tokens;
  const int64_t rows = max_q * group;
  p.mt = group <= 16 && (rows <= 16 || rows > 32) ? 1 : 2;
  p.few = group <= 16 * p.mt;
  p.many = rows > 16 * p.mt;
  const int64_t most = (int64_t)b->table_width * c->page_size;
  const int64_t pairs = (int64_t)(b->num_seqs > 0 ? b->num_seqs : 1) * c->n_kv_heads;
  int64_t splits = (2048 + pairs - 1) / pairs;
  const int64_t cap = (most + 127) / 128;
  splits = splits < cap ? splits : cap;
  splits = splits < 256 ? splits : 256;
  p.splits = (int)(splits > 1 ? splits : 1);
  p.row_stride = (int)(rows < 16 * p.mt ? rows : 16 * p.mt);
  p.part_rows = p.few && p.splits > 1 ? pairs * p.splits * p.row_stride : 0;
  if (p.many) {
    p.items = b->tokens * group / kManyRows + b->num_seqs;
    const int64_t blocks = p.items * c->n_kv_heads;
    int64_t sp = blocks < 256 ? 512 / blocks : 1;
    const int64_t most_sp = (most + 511) / 512;
    sp = sp < most_sp ? sp : most_sp;
    p.many_splits = (int)(sp > 1 ? sp : 1);
    p.many_part_rows = p.many_splits > 1 ? blocks * p.many_splits * kManyRows : 0;
  }
  return p;
}

int64_t round256(int64_t v) { return (v + 255) / 256 * 256; }

// The two kernels run one after the other, each with its join: they share the workspace.
int64_t part_rows_of(const Plan& p) { return p.part_rows > p.many_part_rows ? p.part_rows : p.many_part_rows; }
int64_t workspace_of(const Plan& p, int D) { return round256(part_rows_of(p) * D * 4) + round256(part_rows_of(p) * 8); }

template <int DT, int D>
void launch(AttnArgs& a, const Plan& p, hipStream_t st) {
  const int64_t units = p.few ? (int64_t)a.seqs * a.hk * a.splits : 0, guards = (a.tokens + 255) / 256;
  const dim3 grid = linear_grid(units + guards);
  if (p.mt == 1) kv_attn_few_kernel<DT, D, 1><<<grid, 256, 0, st>>>(a, units, guards);
  else kv_attn_few_kernel<DT, D, 2><<<grid, 256, 0, st>>>(a, units, guards);
  if (p.part_rows) {
    const int64_t rows = (int64_t)a.seqs * a.hk * a.row_stride;
    kv_attn_join_kernel<DT, D><<<linear_grid((rows + 3) / 4), 256, 0, st>>>(a, rows);
  }
  if (!p.many) return;
  a.splits = p.many_splits;
  constexpr int KT = D == 256 ? 32 : 64;
  kv_attn_many_kernel<DT, D, KT><<<linear_grid(p.items * a.hk * a.splits), 256, 0, st>>>(a, p.items);
  if (p.many_part_rows)
    kv_attn_many_join_kernel<DT, D, KT><<<linear_grid(p.items * a.hk * (kManyRows / 4)), 256, 0, st>>>(a, p.items);
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
  a.tokens = b->tokens, a.table_stride = b->table_stride, a.num_pages = c->num_pages;
  a.stride_t = d->q_stride_t, a.stride_h = d->q_stride_h;
  a.seqs = b->num_seqs, a.hq = d->n_q_heads, a.hk = c->n_kv_heads, a.group = d->n_q_heads / c->n_kv_heads;
  a.page_log2 = log2_of(c->page_size), a.table_width = b->table_width;
  a.max_q = d->max_q_len;
  a.causal = d->causal != 0, a.window = d->window;
  a.splits = p.splits, a.row_stride = p.row_stride, a.few_rows = p.few ? 16 * p.mt : 0;
  a.vec = (reinterpret_cast<uintptr_t>(q) & 15) == 0 && d->q_stride_t % 8 == 0 && d->q_stride_h % 8 == 0;
  a.scale2 = d->scale * 1.44269504088896341f;
  if (d->dtype == PDM_BF16) launch_dt<PDM_BF16>(a, c->head_dim, p, stream);
  else launch_dt<PDM_F16>(a, c->head_dim, p, stream);
  PDM_CHECK_LAUNCH();
  return PDM_OK;
}
