// Norm of every query and key head and the position rotation in one pass, and its backward pass.
//
// For the row x [D] of one (token, head), with r = (mean(x^2) + eps)^(-1/2) and n = x r w (n = x where there
// is no weight w), and the pairs (a, b) of the first R elements turned by the angle of the token's position:
//   y_a = n_a cos - n_b sin,  y_b = n_b cos + n_a sin                      (elements behind R: y = n)
// Backward, from dy: g = dy turned back, h = g w,
//   dx = r (h - x r mean(h x r)),   dw = sum over tokens and heads of g x r
// in fp32, rounded once.  Both are bound by HBM: 2 and 3 times the tensors' bytes.  Lane groups of D / 16 lanes take rows, a
// row's 16 elements a lane in registers from its one load to its one store: 8,192 tokens of 32 + 8 heads of 128 in bf16 36 us
// (4.7 TB/s; a copy reaches 5.2), 16 tokens 3.2 us.  With the backward pass, 24,259 tokens of 6 + 6 heads of 64 18.6 + 32.9 +
// 3.9 us (4.0 and 3.4 TB/s, sums of dw), 16,384 tokens of 24 + 6 heads of 128 in fp16 52.3 + 81.2 + 4.0 us (4.8 and 4.6 TB/s).
#include "kv_common.h"

namespace pdm {
namespace {

struct RopeArgs {
  const void* x;            // rows of one part (q or k): element (t, h, d) at t * stride_t + h * stride_h + d
  const float* w;           // [D] or null
  void* y;                  // contiguous [T, H, D] (backward: dx)
  const void* dy;           // backward: contiguous [T, H, D]
  float* partial;           // backward: [blocks of the part][D]
  int64_t stride_t, stride_h;
  uint32_t heads;
  uint32_t rows;            // T * heads
};

struct RopeShared {
  const void* positions;
  const float *cos, *sin;   // [table_rows][R / 2]
  int32_t* err;
  int64_t table_rows;
  int D, R, bits, width;    // width: lanes per row, a power of two >= D / 16
  float eps;
};

// A block walks rows block, block + blocks, ... (in units of its lane groups) of its part; the weight is read once.
template <int DT, bool NORM, bool INTER, bool VEC>
__global__ void __launch_bounds__(256) rope_fwd_kernel(RopeArgs q, RopeArgs k, uint32_t q_blocks, RopeShared s) {
  const bool is_k = blockIdx.x >= q_blocks;
  const RopeArgs a = is_k ? k : q;
  const uint32_t block = is_k ? blockIdx.x - q_blocks : blockIdx.x;
  const uint32_t blocks = is_k ? gridDim.x - q_blocks : q_blocks;
  const int per_block = 256 / s.width;
  const int j = threadIdx.x & (s.width - 1);
  const bool live = 16 * j < s.D;
  const RowPlace pl = row_place<INTER>(live ? j : 0, s.D, s.R);
  float w[16];
  if (NORM && live) {
    load8f(a.w + pl.lo, w);
    load8f(a.w + pl.hi, w + 8);
  }
  // the block's bound is the same for all its threads: every lane stays for the group sums
  for (uint64_t base = (uint64_t)block * per_block; base < a.rows; base += (uint64_t)blocks * per_block) {
    const uint32_t row = (uint32_t)base + threadIdx.x / s.width;
    const bool ok = live && row < a.rows;
    float v[16], c[8], sn[8];
    bool zero = true;
    if (ok) {
      const uint32_t t = row / a.heads, h = row - t * a.heads;
      const int64_t at = (int64_t)t * a.stride_t + (int64_t)h * a.stride_h;
      load8<DT, VEC>(a.x, at + pl.lo, v);
      load8<DT, VEC>(a.x, at + pl.hi, v + 8);
      const int64_t p = load_position(s.positions, s.bits, t);
      const bool beyond = s.R > 0 && p >= s.table_rows;
      zero = p < 0 || beyond;
      if (beyond && s.err) *s.err = 1;
      if (pl.turned && !zero) {
        load8f(s.cos + p * (s.R / 2) + 8 * j, c);
        load8f(s.sin + p * (s.R / 2) + 8 * j, sn);
      }
    }
    if (NORM) {
      float ss = 0.0f;
      if (ok) {
#pragma unroll
        for (int i = 0; i < 16; ++i) ss = __builtin_fmaf(v[i], v[i], ss);
      }
      ss = group_sum(ss, s.width);
      const float r = 1.0f / sqrtf(ss / (float)s.D + s.eps);
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = v[i] * r * w[i];
    }
    if (!ok) continue;
    if (zero) {
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = 0.0f;
    } else if (pl.turned) {
      rotate16<INTER>(v, c, sn);
    }
    const int64_t out = (int64_t)row * s.D;
    store8<DT>(a.y, out + pl.lo, v);
    store8<DT>(a.y, out + pl.hi, v + 8);
  }
}

// A block walks rows block, block + blocks, ... of its part and leaves one partial sum of dw: no atomics, so that the same
// inputs give the same bits.
template <int DT, bool NORM, bool INTER, bool VEC>
__global__ void __launch_bounds__(256) rope_bwd_kernel(RopeArgs q, RopeArgs k, uint32_t q_blocks, RopeShared s) {
  __shared__ float red[256 * 16];
  const bool is_k = blockIdx.x >= q_blocks;
  const RopeArgs a = is_k ? k : q;
  const uint32_t block = is_k ? blockIdx.x - q_blocks : blockIdx.x;
  const uint32_t blocks = is_k ? gridDim.x - q_blocks : q_blocks;
  const int per_block = 256 / s.width;
  const int j = threadIdx.x & (s.width - 1);
  const bool live = 16 * j < s.D;
  const RowPlace pl = row_place<INTER>(live ? j : 0, s.D, s.R);
  float w[16], dw[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) dw[i] = 0.0f;
  if (NORM && live) {
    load8f(a.w + pl.lo, w);
    load8f(a.w + pl.hi, w + 8);
  }
  // the block's bound is the same for all its threads: every lane stays for the group sums
  for (uint64_t base = (uint64_t)block * per_block; base < a.rows; base += (uint64_t)blocks * per_block) {
    const uint32_t row = (uint32_t)base + threadIdx.x / s.width;
    const bool ok = live && row < a.rows;
    float x[16], g[16];
    bool zero = true;
    if (ok) {
      const uint32_t t = row / a.heads, h = row - t * a.heads;
      const int64_t at = (int64_t)t * a.stride_t + (int64_t)h * a.stride_h, out = (int64_t)row * s.D;
      load8<DT, VEC>(a.dy, out + pl.lo, g);
      load8<DT, VEC>(a.dy, out + pl.hi, g + 8);
      if (NORM) {
        load8<DT, VEC>(a.x, at + pl.lo, x);
        load8<DT, VEC>(a.x, at + pl.hi, x + 8);
      }
      const int64_t p = load_position(s.positions, s.bits, t);
      zero = p < 0 || (s.R > 0 && p >= s.table_rows);
      if (pl.turned && !zero) {
        float c[8], sn[8];
        load8f(s.cos + p * (s.R / 2) + 8 * j, c);
        load8f(s.sin + p * (s.R / 2) + 8 * j, sn);
#pragma unroll
        for (int i = 0; i < 8; ++i) sn[i] = -sn[i];
        rotate16<INTER>(g, c, sn);
      }
    }
    if (NORM) {
      float ss = 0.0f, hx = 0.0f;
      if (ok) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          ss = __builtin_fmaf(x[i], x[i], ss);
          hx = __builtin_fmaf(g[i] * w[i], x[i], hx);
        }
      }
      ss = group_sum(ss, s.width);
      hx = group_sum(hx, s.width);
      if (ok) {
        const float r = 1.0f / sqrtf(ss / (float)s.D + s.eps);
        const float m = hx / (float)s.D * r * r;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float gi = g[i];
          if (!zero) dw[i] = __builtin_fmaf(gi, x[i] * r, dw[i]);
          g[i] = r * (gi * w[i] - x[i] * m);
        }
      }
    }
    if (ok) {
      if (zero) {
#pragma unroll
        for (int i = 0; i < 16; ++i) g[i] = 0.0f;
      }
      const int64_t out = (int64_t)row * s.D;
      store8<DT>(a.y, out + pl.lo, g);
      store8<DT>(a.y, out + pl.hi, g + 8);
    }
  }
  if (NORM) {
    // red[element][group]: the groups of a block in a fixed order
#pragma unroll
    for (int i = 0; i < 16; ++i) red[(j * 16 + i) * per_block + threadIdx.x / s.width] = dw[i];
    __syncthreads();
    for (int e = threadIdx.x; e < s.width * 16; e += 256) {
      const int jj = e >> 4, i = e & 15;
      if (16 * jj >= s.D) continue;
      float sum = 0.0f;
      for (int g2 = 0; g2 < per_block; ++g2) sum += red[e * per_block + g2];
      const RowPlace p2 = row_place<INTER>(jj, s.D, s.R);
      a.partial[(int64_t)block * s.D + (i < 8 ? p2.lo + i : p2.hi + i - 8)] = sum;
    }
  }
}

// dw[d] = sum over blocks of partial[block][d], in one fixed order: 32 columns and 32 runs of blocks a workgroup.
__global__ void __launch_bounds__(1024) rope_dw_kernel(const float* pq, const float* pk, uint32_t nq, uint32_t nk, int D,
                                                       float* dwq, float* dwk) {
  __shared__ float red[32][33];
  const float* p = blockIdx.y ? pk : pq;
  float* out = blockIdx.y ? dwk : dwq;
  const uint32_t n = blockIdx.y ? nk : nq;
  if (!out) return;
  const int c = threadIdx.x & 31, g = threadIdx.x >> 5;
  const int d = blockIdx.x * 32 + c;
  float sum = 0.0f;
  if (d < D) {
#pragma unroll 8
    for (uint32_t b = g; b < n; b += 32) sum += p[(int64_t)b * D + d];
  }
  red[g][c] = sum;
  __syncthreads();
  if (g == 0 && d < D) {
    float total = 0.0f;
    for (int i = 0; i < 32; ++i) total += red[i][c];
    out[d] = total;
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

int lanes_per_row(int D) {
  int w = 1;
  while (w * 16 < D) w <<= 1;
  return w;
}

constexpr int64_t kFwdBlocks = 4096;   // of both parts: 8,192 tokens of 32 + 8 heads of 128 37 us with 1,024 to 8,192, 40 with all
constexpr uint32_t kBwdBlocks = 1024;  // blocks of one part in the backward pass, each with a partial sum of dw

uint32_t bwd_blocks(int64_t rows, int D) {
  const int64_t per = 256 / lanes_per_row(D);
  const int64_t b = (rows + per - 1) / per;
  return (uint32_t)(b < kBwdBlocks ? b : kBwdBlocks);
}

int check(const char* fn, const pdm_qk_rope_desc* d) {
  auto bad = [&](const char* m) {
    set_error(std::string(fn) + ": " + m);
    return (int)PDM_ERR_INVALID;
  };
  if (!d) return bad("null descriptor");
  if (d->tokens < 0 || d->n_q_heads < 0 || d->n_k_heads < 0) return bad("negative sizes");
  if (d->head_dim < 16 || d->head_dim > 1024 || d->head_dim % 16) return bad("head_dim must be a multiple of 16 in [16, 1024]");
  if (d->rotary_dim < 0 || d->rotary_dim > d->head_dim || d->rotary_dim % 16) return bad("rotary_dim must be a multiple of 16 in [0, head_dim]");
  if (d->dtype != PDM_F32 && d->dtype != PDM_F16 && d->dtype != PDM_BF16) return bad("dtype must be F32, F16 or BF16");
  if (d->position_bits != 32 && d->position_bits != 64) return bad("position_bits must be 32 or 64");
  if (d->table_rows < 0) return bad("negative table_rows");
  if (!(d->eps >= 0)) return bad("eps must not be negative");
  const int64_t heads = d->n_q_heads > d->n_k_heads ? d->n_q_heads : d->n_k_heads;
  if (heads > (1 << 20) || d->tokens > (int64_t(1) << 31) || d->tokens * heads >= (int64_t(1) << 31))
    return bad("tokens * heads must be below 2^31");
  return PDM_OK;
}

RopeShared shared_of(const pdm_qk_rope_desc* d, const void* positions, const float* cos, const float* sin, int32_t* err) {
  return RopeShared{positions, cos, sin, err, d->table_rows, d->head_dim, d->rotary_dim, d->position_bits,
                    lanes_per_row(d->head_dim), d->eps};
}

template <int DT, bool NORM, bool INTER, bool VEC>
void launch_fwd(const RopeArgs& q, const RopeArgs& k, const RopeShared& s, hipStream_t st) {
  const int64_t per = 256 / s.width;
  auto blocks = [&](const RopeArgs& x) {
    const int64_t b = ((int64_t)x.rows + per - 1) / per, most = kFwdBlocks * (int64_t)x.rows / ((int64_t)q.rows + k.rows) + 1;
    return (uint32_t)(b < most ? b : most);
  };
  const uint32_t nq = blocks(q), nk = blocks(k);
  rope_fwd_kernel<DT, NORM, INTER, VEC><<<nq + nk, 256, 0, st>>>(q, k, nq, s);
}

template <int DT, bool NORM, bool INTER, bool VEC>
void launch_bwd(const RopeArgs& q, const RopeArgs& k, const RopeShared& s, hipStream_t st) {
  const uint32_t nq = bwd_blocks(q.rows, s.D), nk = bwd_blocks(k.rows, s.D);
  rope_bwd_kernel<DT, NORM, INTER, VEC><<<nq + nk, 256, 0, st>>>(q, k, nq, s);
}

template <bool BWD, int DT, bool NORM, bool INTER>
void launch_vec(bool vec, const RopeArgs& q, const RopeArgs& k, const RopeShared& s, hipStream_t st) {
  if constexpr (BWD) {
    if (vec) launch_bwd<DT, NORM, INTER, true>(q, k, s, st);
    else launch_bwd<DT, NORM, INTER, false>(q, k, s, st);
  } else {
    if (vec) launch_fwd<DT, NORM, INTER, true>(q, k, s, st);
    else launch_fwd<DT, NORM, INTER, false>(q, k, s, st);
  }
}

template <bool BWD, int DT>
void launch_dt(bool norm, bool inter, bool vec, const RopeArgs& q, const RopeArgs& k, const RopeShared& s, hipStream_t st) {
  if (norm) {
    if (inter) launch_vec<BWD, DT, true, true>(vec, q, k, s, st);
    else launch_vec<BWD, DT, true, false>(vec, q, k, s, st);
  } else {
    if (inter) launch_vec<BWD, DT, false, true>(vec, q, k, s, st);
    else launch_vec<BWD, DT, false, false>(vec, q, k, s, st);
  }
}

template <bool BWD>
void launch(int dt, bool norm, bool inter, bool vec, const RopeArgs& q, const RopeArgs& k, const RopeShared& s,
            hipStream_t st) {
  if (q.rows + (uint64_t)k.rows == 0) return;
  if (dt == PDM_F32) launch_dt<BWD, PDM_F32>(norm, inter, vec, q, k, s, st);
  else if (dt == PDM_F16) launch_dt<BWD, PDM_F16>(norm, inter, vec, q, k, s, st);
  else launch_dt<BWD, PDM_BF16>(norm, inter, vec, q, k, s, st);
}

// Rows that 16-byte loads reach: base address, strides and (fp32 or 16-bit) pieces of 8 elements.
bool vec_ok(const pdm_qk_rope_desc* d, const void* x, int64_t st, int64_t sh, uint32_t rows) {
  const int64_t unit = d->dtype == PDM_F32 ? 4 : 8;
  return rows == 0 || (aligned16(x) && st % unit == 0 && sh % unit == 0);
}

}  // namespace
}  // namespace pdm

using namespace pdm;

extern "C" int pdm_qk_norm_rope_fwd(const pdm_qk_rope_desc* d, const void* q, const void* k, const void* positions,
                                    const float* cos, const float* sin, const float* q_weight, const float* k_weight,
                                    void* q_out, void* k_out, int32_t* err_flag, pdm_stream_t stream) {
  clear_error();
  if (int e = check(__func__, d)) return e;
  const uint32_t rq = (uint32_t)(d->tokens * d->n_q_heads), rk = (uint32_t)(d->tokens * d->n_k_heads);
  PDM_CHECK_ARG((!rq || (q && q_out)) && (!rk || (k && k_out)), "null q / k");
  PDM_CHECK_ARG(!d->tokens || positions, "null positions");
  PDM_CHECK_ARG(!d->rotary_dim || (cos && sin), "null cos / sin");
  PDM_CHECK_ARG(!rq || !rk || (!q_weight == !k_weight), "weights for both of q and k, or for neither");
  PDM_CHECK_ARG(aligned16(q_out) && aligned16(k_out) && aligned16(cos) && aligned16(sin) && aligned16(q_weight) &&
                    aligned16(k_weight), "outputs, cos, sin and weights must be 16-byte aligned");
  const RopeArgs aq{q, q_weight, q_out, nullptr, nullptr, d->q_stride_t, d->q_stride_h, (uint32_t)d->n_q_heads, rq};
  const RopeArgs ak{k, k_weight, k_out, nullptr, nullptr, d->k_stride_t, d->k_stride_h, (uint32_t)d->n_k_heads, rk};
  const bool vec = vec_ok(d, q, d->q_stride_t, d->q_stride_h, rq) && vec_ok(d, k, d->k_stride_t, d->k_stride_h, rk);
  launch<false>(d->dtype, (rq ? q_weight : k_weight) != nullptr, d->interleaved != 0, vec, aq, ak,
                shared_of(d, positions, cos, sin, err_flag), stream);
  PDM_CHECK_LAUNCH();
  return PDM_OK;
}

extern "C" int64_t pdm_qk_norm_rope_bwd_workspace_size(const pdm_qk_rope_desc* d) {
  clear_error();
  if (int e = check(__func__, d)) return e;
  return (int64_t)(bwd_blocks(d->tokens * d->n_q_heads, d->head_dim) + bwd_blocks(d->tokens * d->n_k_heads, d->head_dim)) *
         d->head_dim * 4;
}

extern "C" int pdm_qk_norm_rope_bwd(const pdm_qk_rope_desc* d, const void* q, const void* k, const void* positions,
                                    const float* cos, const float* sin, const float* q_weight, const float* k_weight,
                                    const void* grad_q_out, const void* grad_k_out, void* grad_q, void* grad_k,
                                    float* grad_q_weight, float* grad_k_weight, void* workspace, int64_t workspace_bytes,
                                    pdm_stream_t stream) {
  clear_error();
  if (int e = check(__func__, d)) return e;
  const uint32_t rq = (uint32_t)(d->tokens * d->n_q_heads), rk = (uint32_t)(d->tokens * d->n_k_heads);
  const bool norm = (rq ? q_weight : rk ? k_weight : q_weight ? q_weight : k_weight) != nullptr;  // (no rows: zero sums)
  PDM_CHECK_ARG((!rq || (grad_q_out && grad_q && (!norm || q))) && (!rk || (grad_k_out && grad_k && (!norm || k))),
                "null q / k or gradients");
  PDM_CHECK_ARG(!d->tokens || positions, "null positions");
  PDM_CHECK_ARG(!d->rotary_dim || (cos && sin), "null cos / sin");
  PDM_CHECK_ARG(!rq || !rk || (!q_weight == !k_weight), "weights for both of q and k, or for neither");
  PDM_CHECK_ARG(aligned16(grad_q) && aligned16(grad_k) && aligned16(cos) && aligned16(sin) && aligned16(q_weight) &&
                    aligned16(k_weight) && aligned16(workspace), "gradients, cos, sin, weights and workspace must be 16-byte aligned");
  const int64_t need = pdm_qk_norm_rope_bwd_workspace_size(d);
  if (norm && (workspace_bytes < need || (!workspace && need > 0))) {
    set_error(std::string(__func__) + ": workspace of " + std::to_string(need) + " bytes needed");
    return PDM_ERR_WORKSPACE;
  }
  const uint32_t nq = bwd_blocks(rq, d->head_dim), nk = bwd_blocks(rk, d->head_dim);
  float* pq = static_cast<float*>(workspace);
  float* pk = norm ? pq + (int64_t)nq * d->head_dim : nullptr;
  const RopeArgs aq{q, q_weight, grad_q, grad_q_out, pq, d->q_stride_t, d->q_stride_h, (uint32_t)d->n_q_heads, rq};
  const RopeArgs ak{k, k_weight, grad_k, grad_k_out, pk, d->k_stride_t, d->k_stride_h, (uint32_t)d->n_k_heads, rk};
  const bool vec = vec_ok(d, q, d->q_stride_t, d->q_stride_h, norm ? rq : 0) &&
                   vec_ok(d, k, d->k_stride_t, d->k_stride_h, norm ? rk : 0) && aligned16(grad_q_out) && aligned16(grad_k_out);
  launch<true>(d->dtype, norm, d->interleaved != 0, vec, aq, ak, shared_of(d, positions, cos, sin, nullptr), stream);
  if (norm && (grad_q_weight || grad_k_weight)) {
    rope_dw_kernel<<<dim3((d->head_dim + 31) / 32, 2), 1024, 0, stream>>>(pq, pk, nq, nk, d->head_dim,
                                                                          grad_q_weight, grad_k_weight);
  }
  PDM_CHECK_LAUNCH();
  return PDM_OK;
}
