// Attention of new tokens over an 8-bit paged cache: one wave per (query row, head).
#include "kv_common.h"

namespace pdm {
namespace {

struct AttnArgs {
  const void* q;
  void* out;
  float* lse;
  const uint8_t *k_codes, *v_codes;
  const float *k_scale, *v_scale;
  const int32_t *cu, *table, *lens;
  int32_t* err;
  int64_t tokens, table_stride, num_pages, stride_t, stride_h;
  int32_t seqs, hq, hk, D, page_log2, table_width, max_q, causal, window;
  float scale;
};

__device__ __forceinline__ float e4m3_to_f32(uint32_t c) { return __builtin_amdgcn_cvt_f32_fp8((int)c, 0); }

template <int DT>
__global__ void __launch_bounds__(64) kv_attn_row_kernel(AttnArgs a) {
  __shared__ float qs[256];
  const int64_t unit = linear_block();
  const int64_t t = unit / a.hq;
  if (t >= a.tokens) return;
  const int h = (int)(unit - t * a.hq), kh = h / (a.hq / a.hk);
  const int lane = threadIdx.x;
  const int b = find_sequence(a.seqs, t, [&](int i) { return (int64_t)a.cu[i]; });
  int64_t lo = 0, hi = 0;
  if (a.seqs > 0 && t >= a.cu[b] && t < a.cu[b + 1]) {
    const int64_t n = (int64_t)a.cu[b + 1] - a.cu[b];
    int64_t len = a.lens[b];
    if (a.cu[b] < 0 || a.cu[b + 1] > a.tokens || n > a.max_q || n > len) {
      if (a.err) *a.err = 1;
    } else {
      const int64_t p = len - n + (t - a.cu[b]);
      hi = a.causal ? p + 1 : len;
      if (hi > len) hi = len;
      lo = a.window > 0 && p - a.window + 1 > 0 ? p - a.window + 1 : 0;
      if (hi > (int64_t)a.table_width << a.page_log2) {
        hi = (int64_t)a.table_width << a.page_log2;
        if (a.err) *a.err = 1;
      }
    }
  }
  for (int d = lane; d < a.D; d += 64) {
    const int64_t at = t * a.stride_t + h * a.stride_h + d;
    const uint32_t u = static_cast<const uint16_t*>(a.q)[at];
    qs[d] = DT == PDM_BF16 ? bf16_bits_to_f32(u) : f16_bits_to_f32(u);
  }
  __syncthreads();
  float m = -__builtin_inff(), l = 0.0f, acc[4] = {0, 0, 0, 0};
  for (int64_t base = lo; base < hi; base += 64) {
    const int64_t j = base + lane;
    float s = -__builtin_inff();
    int64_t row = -1;  // (page * heads + head) * page_size + slot
    float vs = 0.0f;
    if (j < hi) {
      const int64_t id = a.table[(int64_t)b * a.table_stride + (j >> a.page_log2)];
      if (id < 0 || id >= a.num_pages) {
        if (a.err) *a.err = 1;
      } else {
        const int64_t entry = id * a.hk + kh;
        row = (entry << a.page_log2) + (j & ((1 << a.page_log2) - 1));
        float dot = 0.0f;
        const uint8_t* kp = a.k_codes + row * a.D;
        for (int d = 0; d < a.D; ++d) dot += qs[d] * e4m3_to_f32(kp[d]);
        s = dot * a.k_scale[entry] * a.scale;
        vs = a.v_scale[entry];
      }
    }
    const float mn = fmaxf(m, group_max(s, 64));
    if (mn == -__builtin_inff() && !__any(s != s)) continue;
    const float f = m == -__builtin_inff() ? 0.0f : expf(m - mn);
    const float p = row >= 0 ? expf(s - mn) : 0.0f;
    l = l * f + group_sum(p, 64);
    for (int i = 0; i < 4; ++i) acc[i] *= f;
    m = mn;
    for (int x = 0; x < 64; ++x) {
      const int64_t r = __shfl(row, x);
      const float px = __shfl(p, x), vx = __shfl(vs, x);
      if (r < 0) continue;
      for (int i = 0; i * 64 < a.D; ++i) acc[i] += px * (vx * e4m3_to_f32(a.v_codes[r * a.D + i * 64 + lane]));
    }
  }
  for (int i = 0; i * 64 < a.D; ++i) {
    const float o = l != 0.0f ? acc[i] / l : 0.0f;
    static_cast<uint16_t*>(a.out)[(t * a.hq + h) * a.D + i * 64 + lane] =
        (uint16_t)(DT == PDM_BF16 ? f32_to_bf16_bits(o) : f32_to_f16_bits(o));
  }
  if (lane == 0 && a.lse) a.lse[t * a.hq + h] = l != 0.0f ? m + logf(l) : -__builtin_inff();
}

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

}  // namespace
}  // namespace pdm

using namespace pdm;

extern "C" int64_t pdm_kv_attention_workspace_size(const pdm_kv_attention_desc* d, const pdm_kv_cache* c,
                                                   const pdm_kv_batch* b) {
  clear_error();
  if (int e = check(__func__, d, c, b)) return e;
  return 0;
}

extern "C" int pdm_kv_attention_fwd(const pdm_kv_attention_desc* d, const pdm_kv_cache* c, const pdm_kv_batch* b,
                                    const void* q, void* out, float* lse, void* workspace, int64_t workspace_bytes,
                                    int32_t* err_flag, pdm_stream_t stream) {
  clear_error();
  if (int e = check(__func__, d, c, b)) return e;
  if (b->tokens == 0) return PDM_OK;
  PDM_CHECK_ARG(q && out, "null q / out");
  PDM_CHECK_ARG((reinterpret_cast<uintptr_t>(out) & 15) == 0, "out must be 16-byte aligned");
  AttnArgs a{};
  a.q = q, a.out = out, a.lse = lse;
  a.k_codes = c->k_codes, a.v_codes = c->v_codes, a.k_scale = c->k_scale, a.v_scale = c->v_scale;
  a.cu = b->cu_seqlens, a.table = b->page_table, a.lens = b->seq_lens, a.err = err_flag;
  a.tokens = b->tokens, a.table_stride = b->table_stride, a.num_pages = c->num_pages;
  a.stride_t = d->q_stride_t, a.stride_h = d->q_stride_h;
  a.seqs = b->num_seqs, a.hq = d->n_q_heads, a.hk = c->n_kv_heads, a.D = c->head_dim;
  a.page_log2 = log2_of(c->page_size), a.table_width = b->table_width, a.max_q = d->max_q_len;
  a.causal = d->causal != 0, a.window = d->window, a.scale = d->scale;
  const dim3 grid = linear_grid(b->tokens * d->n_q_heads);
  if (d->dtype == PDM_BF16) kv_attn_row_kernel<PDM_BF16><<<grid, 64, 0, stream>>>(a);
  else kv_attn_row_kernel<PDM_F16><<<grid, 64, 0, stream>>>(a);
  PDM_CHECK_LAUNCH();
  return PDM_OK;
}
