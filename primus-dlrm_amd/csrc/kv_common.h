// Device helpers of the cached-attention operators (qk_rope.hip, kv_append.hip, kv_attention.hip): rows of
// a head as 16 elements per lane, the position rotation, the e4m3 conversions and the page lookups.
#pragma once

#include "mfma_common.h"

namespace pdm {

// ---- a head's row, 16 elements per lane -------------------------------------
// Lane j of a row's group holds two pieces of 8 elements, so that a rotated pair never leaves its lane:
//   halves:      pieces 8j and R/2 + 8j for 8j < R/2 (pairs (i, i + R/2)); behind the rotated part
//                R + 8m and R + 8m + (D - R)/2, m = j - R/16
//   neighbours:  pieces 16j and 16j + 8 (pairs (2i, 2i + 1))
// In both the pairs of lane j < R/16 use entries 8j .. 8j + 7 of the position's cos / sin row.
struct RowPlace {
  int lo, hi;    // first element of the two pieces
  bool turned;   // inside the rotated part
};

template <bool INTER>
__device__ __forceinline__ RowPlace row_place(int j, int D, int R) {
  RowPlace p;
  p.turned = 16 * j < R;
  if (INTER) {
    p.lo = 16 * j;
    p.hi = p.lo + 8;
  } else if (p.turned) {
    p.lo = 8 * j;
    p.hi = p.lo + R / 2;
  } else {
    p.lo = R + 8 * (j - R / 16);
    p.hi = p.lo + (D - R) / 2;
  }
  return p;
}

// Eight elements of dtype DT (PDM_F32 / PDM_F16 / PDM_BF16) as they are stored, in two (fp32) or one register quads; VEC:
// 16-byte aligned.
template <int DT, bool VEC>
__device__ __forceinline__ void load8_raw(const void* base, int64_t at, u32x4_t* w) {
  if constexpr (DT == PDM_F32) {
    const uint32_t* p = static_cast<const uint32_t*>(base) + at;
    if constexpr (VEC) {
      w[0] = *reinterpret_cast<const u32x4_t*>(p), w[1] = *reinterpret_cast<const u32x4_t*>(p + 4);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) w[0][i] = p[i], w[1][i] = p[4 + i];
    }
  } else {
    const uint16_t* p = static_cast<const uint16_t*>(base) + at;
    if constexpr (VEC) {
      w[0] = *reinterpret_cast<const u32x4_t*>(p);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) w[0][i] = uint32_t(p[2 * i]) | uint32_t(p[2 * i + 1]) << 16;
    }
  }
}

template <int DT>
__device__ __forceinline__ void raw_to_float(const u32x4_t* w, float* v) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (DT == PDM_F32) {
      v[i] = __uint_as_float(w[0][i]), v[4 + i] = __uint_as_float(w[1][i]);
    } else if constexpr (DT == PDM_BF16) {
      v[2 * i] = __uint_as_float(w[0][i] << 16);
      v[2 * i + 1] = __uint_as_float(w[0][i] & 0xffff0000u);
    } else {
      v[2 * i] = f16_bits_to_f32(w[0][i] & 0xffffu);
      v[2 * i + 1] = f16_bits_to_f32(w[0][i] >> 16);
    }
  }
}

// The same as fp32.
template <int DT, bool VEC>
__device__ __forceinline__ void load8(const void* base, int64_t at, float* v) {
  u32x4_t w[2];
  load8_raw<DT, VEC>(base, at, w);
  raw_to_float<DT>(w, v);
}

// Eight fp32 values rounded once to dtype DT; the address is 16-byte aligned.
template <int DT>
__device__ __forceinline__ void store8(void* base, int64_t at, const float* v) {
  if constexpr (DT == PDM_F32) {
    float* p = static_cast<float*>(base) + at;
    *reinterpret_cast<f32x4_t*>(p) = f32x4_t{v[0], v[1], v[2], v[3]};
    *reinterpret_cast<f32x4_t*>(p + 4) = f32x4_t{v[4], v[5], v[6], v[7]};
  } else {
    u32x4_t w;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (DT == PDM_BF16) w[i] = pack_bf16x2(v[2 * i], v[2 * i + 1]);
      else w[i] = f32_to_f16_bits(v[2 * i]) | f32_to_f16_bits(v[2 * i + 1]) << 16;
    }
    *reinterpret_cast<u32x4_t*>(static_cast<uint16_t*>(base) + at) = w;
  }
}

__device__ __forceinline__ void load8f(const float* p, float* v) {
  const f32x4_t a = *reinterpret_cast<const f32x4_t*>(p), b = *reinterpret_cast<const f32x4_t*>(p + 4);
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = a[i], v[i + 4] = b[i];
}

// The rotation of a lane's 16 elements (F: float or double) by the angles of cos / sin.
template <bool INTER, typename F>
__device__ __forceinline__ void rotate16(F* v, const float* c, const float* s) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int a = INTER ? 2 * i : i, b = INTER ? 2 * i + 1 : i + 8;
    const F x = v[a], y = v[b];
    v[a] = x * c[i] - y * s[i];
    v[b] = y * c[i] + x * s[i];
  }
}

// Sum / max over the `width` lanes of a row's group (a power of two <= 64), in every lane of it.
__device__ __forceinline__ float group_sum(float v, int width) {
  for (int o = 1; o < width; o <<= 1) v += __shfl_xor(v, o);
  return v;
}
__device__ __forceinline__ float group_max(float v, int width) {
  for (int o = 1; o < width; o <<= 1) v = fmaxf(v, __shfl_xor(v, o));
  return v;
}

// A workgroup barrier that orders LDS alone: global loads stay in flight across it (__syncthreads waits for them).
__device__ __forceinline__ void lds_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// ---- positions ---------------------------------------------------------------
__device__ __forceinline__ int64_t load_position(const void* positions, int bits, int64_t t) {
  return bits == 64 ? static_cast<const int64_t*>(positions)[t] : (int64_t)static_cast<const int32_t*>(positions)[t];
}

// ---- e4m3 codes under a power-of-two scale -------------------------------------
// A page of one head has the scale 2^e with the smallest e for which no value exceeds 448 * 2^e, held within
// [-117, 119]: every code times its scale is then zero or a normal bf16 value, exactly.
constexpr int kScaleExpMin = -117, kScaleExpMax = 119;
constexpr float kE4m3Max = 448.0f;

__device__ __forceinline__ int scale_exponent(float amax) {
  // 448 = 1.75 * 2^8: amax = f * 2^x with 1 <= f < 2 needs e = x - 8, one more where f > 1.75
  const uint32_t u = __float_as_uint(amax);
  const int e = (int)(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  return e < kScaleExpMin ? kScaleExpMin : e > kScaleExpMax ? kScaleExpMax : e;  // zero and denormals: the smallest
}
__device__ __forceinline__ float exp2_int(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }
__device__ __forceinline__ int scale_exponent_of(float scale) { return (int)((__float_as_uint(scale) >> 23) & 0xffu) - 127; }

// Four values (already divided by the scale) to e4m3, nearest even; NaN and infinities become the NaN code, as does what is
// beyond 448 (after rounding: 464 and more).
__device__ __forceinline__ uint32_t e4m3x4(const float* v) {
  uint32_t w = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], (int)w, true);
}

// A finite value beyond 448 (under the largest scale alone) saturates.
__device__ __forceinline__ float e4m3_saturated(float v) {
  return fabsf(v) < __builtin_inff() ? __builtin_amdgcn_fmed3f(v, -kE4m3Max, kE4m3Max) : v;
}

// ---- sequences -----------------------------------------------------------------
// The sequence whose span of a list of items holds `item`, where sequence b's span begins at first(b), an
// increasing function of b: the last b in [0, n) with first(b) <= item (0 if there is none).  Called by a
// whole wave; 64 entries are looked at per step.
template <typename F>
__device__ __forceinline__ int find_sequence(int n, int64_t item, F first) {
  const int lane = threadIdx.x & 63;
  int lo = 0, len = n;  // the answer lies in [lo, lo + len)
  while (len > 1) {
    const int step = (len + 63) >> 6;
    const int at = lane * step;
    const bool below = at < len && first(lo + at) <= item;
    const unsigned long long m = __ballot(below);
    const int k = m ? 63 - __builtin_clzll(m) : 0;
    lo += k * step;
    len = len - k * step < step ? len - k * step : step;
  }
  return lo;
}

// ---- host checks ----------------------------------------------------------------
inline int log2_of(int v) {
  int l = 0;
  while ((1 << l) < v) ++l;
  return l;
}

inline int check_cache(const char* fn, const pdm_kv_cache* c, const pdm_kv_batch* b) {
  auto bad = [&](const char* m) {
    set_error(std::string(fn) + ": " + m);
    return (int)PDM_ERR_INVALID;
  };
  if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256) return bad("head_dim must be 64, 128 or 256");
  if (c->page_size != 16 && c->page_size != 32 && c->page_size != 64 && c->page_size != 128)
    return bad("page_size must be 16, 32, 64 or 128");
  if (c->n_kv_heads < 1 || c->n_kv_heads > 1024) return bad("n_kv_heads must lie in [1, 1024]");
  if (c->num_pages < 0 || c->num_pages > 0x7fffffff) return bad("num_pages must lie in [0, 2^31)");
  if (b->tokens < 0 || b->num_seqs < 0 || b->table_width < 0 || b->table_stride < 0) return bad("negative sizes");
  if (b->tokens >= (int64_t(1) << 31)) return bad("tokens must be below 2^31");
  if (b->num_seqs > (1 << 24)) return bad("num_seqs must not exceed 2^24");
  if ((int64_t)b->table_width * c->page_size > (1 << 30)) return bad("table_width * page_size must not exceed 2^30");
  if (c->num_pages && !(c->k_codes && c->v_codes && c->k_scale && c->v_scale)) return bad("null cache");
  if (((reinterpret_cast<uintptr_t>(c->k_codes) | reinterpret_cast<uintptr_t>(c->v_codes)) & 15) != 0)
    return bad("codes must be 16-byte aligned");
  if (b->num_seqs && !(b->cu_seqlens && b->seq_lens && (b->page_table || b->table_width == 0)))
    return bad("null cu_seqlens, seq_lens or page_table");
  return PDM_OK;
}

}  // namespace pdm
