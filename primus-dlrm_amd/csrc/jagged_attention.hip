// Attention of ragged batches, forward: causal or not, under a window with first tokens that stay visible, with a bias by
// distance.
//
// A workgroup takes 128 queries of one head of one sequence, 32 a wave, and walks the keys in tiles of 64 with the running
// maximum and sum of the softmax.  Both products are transposed, S^T = K Q^T and O^T = V^T P^T: a lane holds scores of one
// query alone, and P^T leaves the first product as the second takes it, when V's rows are read in the same order
// (transposing reads of LDS).
//
// Weights are rounded to the type of the values for the product, half a step of each, as the outputs are; where the gradient
// of a bias is wanted (`rest`), which is a sum of many small differences in 32 bits, they go in as two numbers and what the
// rounding of the outputs left is kept for the backward pass (rest2), with each row's weights in the bias's outer columns (151 -> 158 us
// for the 8,134 tokens of jagged_backward.hip, 132 -> 144 for its sequences on both sides).
//
// Bound by the softmax beside the products: 16,384 tokens, 16 heads on 8, causal and on both sides: heads of 128 1,082 and 2,135 us, 1.02
// and 1.03 PFLOP/s; heads of 64, with as many exponentials for half the products, 685 and 1,229 us, 0.80 and 0.89 (a large
// library product on such a card 1.24).  Under a window of 1,024 the tiles at both of its ends are whole and half used: 8,192 tokens, 32 heads of 128 on 8, 4 sinks: 180 us, 0.72
// PFLOP/s of what is seen.  128 queries a workgroup: 64 would bring every tile twice as often, and 256 leave half of the CUs idle
// in ordinary batches; three waves a SIMD for heads of 64, two for 128, whose sums take 64 registers.
#include "jagged_common.h"

namespace pdm {
namespace {

constexpr int M = 128, KT = 64;

// Weights are exp2 of scores less a reference, which moves only where a weight would pass 2^kRoom.  bf16 holds any power, and its
// values go up to 2^128: the reference lies 30 above the largest score, and 2^22 keys of the largest value do not overflow
// the sums.  fp16 holds weights down to 2^-14 in full, and its values are below 2^16: the reference is a maximum itself.
template <int DT> constexpr float kLift = DT == PDM_BF16 ? 30.0f : 0.0f;
template <int DT> constexpr float kRoom = 8.0f - kLift<DT>;

template <int DT, int D, bool BIAS, bool FINE>
__global__ void __launch_bounds__(256, D == 64 ? 3 : 2) jag_fwd_kernel(JagArgs a, int64_t units) {
  constexpr int KK = D / 16, DD = D / 32;
  __shared__ alignas(1024) char sk[2][KT * Tile<D>::RS];
  __shared__ alignas(1024) char sv[2][KT * Tile<D>::RS];
  __shared__ float sb[2][BIAS ? M + KT : 1];

  const int64_t unit = linear_block();
  if (unit >= units) {
    const int64_t first = (unit - units) * 256;
    if (first >= a.q_tokens && first >= a.seqs) return;
    jag_guard(a, a.cu_q, a.q_tokens, first, [&](int64_t t) {
      clear_row(a.out, t * a.hq * D, a.hq * D);
      if (a.rest) clear_row(a.rest, t * a.hq * D, a.hq * D);
      for (int h = threadIdx.x; h < a.hq; h += 256) {
        if (a.lse) a.lse[t * a.hq + h] = -kInf;
        if (a.stats) a.stats[2 * (t * a.hq + h)] = kNoKeys, a.stats[2 * (t * a.hq + h) + 1] = 0.0f;
        if (FINE && a.outer) a.outer[2 * (t * a.hq + h)] = a.outer[2 * (t * a.hq + h) + 1] = 0.0f;
      }
    });
    return;
  }
  // the query heads of a key head one after the other: with 8 key heads each has its keys in the cache of one XCD
  const int hx = (int)(unit % a.hq), kh = hx % a.hk, head = kh * a.group + hx / a.hk;
  const int64_t place = unit / a.hq;
  JagSeq s;
  int b, r0;
  // later queries see more keys: they begin first
  if (!(a.seqs <= 64 ? jag_ranked_block<M>(a, false, place, s, b, r0) : jag_block<M>(a, a.cu_q, a.items - 1 - place, s, b, r0))) return;

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 31, h = lane >> 5;
  const int off = s.nk - s.nq;
  const JagKeys keys = jag_keys<KT>(a, s, r0, (r0 + M < s.nq ? r0 + M : s.nq) - 1);

  // this lane's query and the keys that it sees: [row_lo, row_lo + row_n) and those below row_first
  const int row = r0 + wave * 32 + c, pos = off + row;
  int row_lo = 0, row_n = 0, row_first = 0;
  const float scale2 = fmaxf(fabsf(a.scale2), 0x1p-126f);  // not zero: a hidden score times it stays -inf
  if (row < s.nq) {
    const int hi = a.causal && pos + 1 < s.nk ? (pos + 1 > 0 ? pos + 1 : 0) : s.nk;
    row_lo = a.window > 0 && pos - a.window + 1 > 0 ? pos - a.window + 1 : 0;
    row_n = hi > row_lo ? hi - row_lo : 0;
    row_first = a.sinks < hi ? a.sinks : hi;
  }
  // of the wave: positions of its first and last query
  const int w0 = r0 + wave * 32, p_first = off + w0, p_last = off + (w0 + 31 < s.nq ? w0 + 31 : s.nq - 1);

  const uint16_t* kp = static_cast<const uint16_t*>(a.k) + s.k0 * a.k_st + kh * a.k_sh;
  const uint16_t* vp = static_cast<const uint16_t*>(a.v) + s.k0 * a.v_st + kh * a.v_sh;
  const float* brow = BIAS ? a.bias + (int64_t)head * (a.bias_last + 1) : nullptr;
  Bring<D, KT> bring_k, bring_v;
  bring_k.init(a.k_st, lane, wave);
  bring_v.init(a.v_st, lane, wave);
  float bias_next = 0.0f;
  const int bias_at = bias_from(a, (int64_t)off + r0 - (KT - 1));
  auto load_k = [&](int t) { bring_k.load(kp, a.k_st, jag_key<KT>(keys, t), s.nk, sk[t & 1], wave); };
  auto load_v = [&](int t) { bring_v.load(vp, a.v_st, jag_key<KT>(keys, t), s.nk, sv[t & 1], wave); };
  auto load_bias = [&](int t) {  // entry x: distance of query r0 + x - 63 from the tile's first key
    if (BIAS && tid < M + KT) bias_next = bias2(a, brow, bias_at - jag_key<KT>(keys, t) + tid);
  };
  auto store_bias = [&](int t) {
    if (BIAS && tid < M + KT) sb[t & 1][tid] = bias_next;
  };

  constexpr f32x16_t zero16 = {0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
  float m = -kInf, l = 0.0f, l_far = 0.0f, l_near = 0.0f;  // FINE: sums of the weights in and behind the bias's last column, before its first
  f32x16_t o[DD];
#pragma unroll
  for (int d = 0; d < DD; ++d) o[d] = zero16;
  const uint32_t row_at = Tile<D>::row_at(lane), col_at = Tile<D>::col_at(lane);

  // of a tile: no query of this wave sees a key; every one sees all keys; of a key: this lane's query sees it
  auto unseen = [&](int key) {
    return w0 >= s.nq || (a.causal && key > p_last) || (a.window > 0 && key + KT - 1 <= p_first - a.window && key >= a.sinks);
  };
  auto all_seen = [&](int key) {
    return key + KT <= s.nk && (!a.causal || key + KT - 1 <= p_first) && (a.window == 0 || key > p_last - a.window || key + KT <= a.sinks);
  };
  // some pair of the workgroup's queries and the tile's keys is not seen (what lies behind the last key comes as zeros)
  const int b_first = off + r0, b_last = off + (r0 + M < s.nq ? r0 + M : s.nq) - 1;
  auto in_part = [&](int key) {
    return (a.causal && key + KT - 1 > b_first) || (a.window > 0 && key <= b_last - a.window && key + KT > a.sinks);
  };
  auto sees = [&](int j) { return (uint32_t)(j - row_lo) < (uint32_t)row_n || j < row_first; };
  bool odd = false, large = false;  // large: scores are multiplied by the scale and rounded, as the reference is

  const int tiles = keys.tiles;
  // the queries come beside the first tile, by way of the second's place
  char* own = (wave < 2 ? sk[1] : sv[1]) + (wave & 1) * 32 * Tile<D>::RS;
  bring_own<D>(static_cast<const uint16_t*>(a.q) + s.q0 * a.q_st + head * a.q_sh, a.q_st, w0, s.nq, own);
  if (tiles > 0) load_k(0), load_v(0), load_bias(0);
  brought();
  u32x4_t q[KK];
#pragma unroll
  for (int kk = 0; kk < KK; ++kk) q[kk] = Tile<D>::rows(own, row_at, 0, kk);
  if (a.scale2 < 0.0f) {  // the scale's sign goes into the queries
#pragma unroll
    for (int kk = 0; kk < KK; ++kk)
#pragma unroll
      for (int e = 0; e < 4; ++e) q[kk][e] ^= 0x80008000u;
  }

  // ---- the steps of a tile ----
  f32x16_t sc[2];
  u32x4_t p[4], rest[4];
  auto scores = [&](int t) __attribute__((always_inline)) {
    if (unseen(jag_key<KT>(keys, t))) return;
    const char* tk = sk[t & 1];
    __builtin_amdgcn_sched_barrier(0);
    sc[0] = zero16, sc[1] = zero16;
#pragma unroll
    for (int kk = 0; kk < KK; ++kk)
#pragma unroll
      for (int x = 0; x < 2; ++x) sc[x] = mfma32<DT>(Tile<D>::rows(tk, row_at, 32 * x, kk), q[kk], sc[x]);
    sched_mfma_ds_pipeline<2 * KK, 8>();
    __builtin_amdgcn_sched_barrier(0);
  };
  auto weights = [&](int t) __attribute__((always_inline)) {
    const int key = jag_key<KT>(keys, t);
    if (unseen(key)) return;
    // Without a bias the scale is left to the exponent's argument.
    float f = scale2;
    if constexpr (BIAS) {
      const float* b = &sb[t & 1][wave * 32 + c + KT - 1 - 4 * h];
      f = 1.0f;
#pragma unroll
      for (int e = 0; e < 32; ++e)  // element e: key 32 (e / 16) + 8 (e / 4 % 4) + e % 4 + 4 h
        sc[e >> 4][e & 15] = __builtin_fmaf(sc[e >> 4][e & 15], scale2, b[-(32 * (e >> 4) + 8 * ((e >> 2) & 3) + (e & 3))]);
    }
    if (!all_seen(key)) {
#pragma unroll
      for (int e = 0; e < 32; ++e)
        sc[e >> 4][e & 15] = sees(key + 4 * h + 32 * (e >> 4) + 8 * ((e >> 2) & 3) + (e & 3)) ? sc[e >> 4][e & 15] : -kInf;
    }
    float top = sc[0][0];
#pragma unroll
    for (int e = 1; e < 32; ++e) top = fmaxf(top, sc[e >> 4][e & 15]);
    top *= f;
    if (__any(top > m + kRoom<DT>)) {
      top = fmaxf(top, __shfl_xor(top, 32));
      const float now = top > m + kRoom<DT> ? top + kLift<DT> : m;  // by row: other rows change nothing
      const float g = now == -kInf ? 1.0f : __builtin_amdgcn_exp2f(m - now);
      m = now;
      l *= g;
      if (FINE) l_far *= g, l_near *= g;
#pragma unroll
      for (int d = 0; d < DD; ++d) o[d] *= g;
      if (!BIAS && __any(fabsf(m) > kLargeScore)) large = true;
    }
    if (!BIAS && large) {  // what rounding left of the largest score would count as 2^32 and more from 2^30 on
#pragma unroll
      for (int e = 0; e < 32; ++e) sc[e >> 4][e & 15] *= f;
      f = 1.0f;
    }
    const float base = m == -kInf ? 0.0f : m;
    float of_tile = 0.0f;
#pragma unroll
    for (int y = 0; y < 4; ++y) {
      float w[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float x = sc[y >> 1][8 * (y & 1) + e];
        w[e] = __builtin_amdgcn_exp2f(BIAS ? x - base : __builtin_fmaf(x, f, -base));
      }
      const float of_keys = ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
      l += of_keys;
      if (FINE) of_tile += of_keys;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        p[y][e] = pack2<DT>(w[2 * e], w[2 * e + 1]);
        if (FINE) rest[y][e] = left2<DT>(w[2 * e], w[2 * e + 1], p[y][e]);
      }
    }
    if constexpr (FINE) {
      // columns of the wave's pairs, but for those of keys ahead or behind the window
      const int from = p_first - key - (KT - 1), to = p_last - key;
      const int first = (a.causal && from < 0 ? 0 : from) - a.bias_start;
      const int last = (a.window > 0 && key >= a.sinks && to >= a.window ? a.window - 1 : to) - a.bias_start;
      float far = first >= a.bias_last ? of_tile : 0.0f, near = last < 0 ? of_tile : 0.0f;
      if ((first < 0 && last >= 0) || (first < a.bias_last && last >= a.bias_last)) {
        const int col0 = pos - a.bias_start - key - 4 * h;
        far = near = 0.0f;
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          const int col = col0 - (32 * (e >> 4) + 8 * ((e >> 2) & 3) + (e & 3));
          uint32_t w = p[e >> 3][e >> 1 & 3], r = rest[e >> 3][e >> 1 & 3];
          asm volatile("" : "+v"(w), "+v"(r));  // else what they were made of is kept for this
          const float x = e & 1 ? hi_of<DT>(w) + hi_of<DT>(r) : lo_of<DT>(w) + lo_of<DT>(r);
          far += col >= a.bias_last ? x : 0.0f;
          near += col < 0 ? x : 0.0f;
        }
      }
      l_far += far, l_near += near;
    }
  };
  auto values = [&](int t) __attribute__((always_inline)) {
    if (unseen(jag_key<KT>(keys, t))) return;
    __builtin_amdgcn_sched_barrier(0);
    add_cols<DT, D, 4, FINE>(o, sv[t & 1], col_at, 0, p, rest);
    __builtin_amdgcn_sched_barrier(0);
  };

#pragma unroll 1
  for (int t = 0; t < tiles; ++t) {
    store_bias(t);
    brought();
    if (in_part(jag_key<KT>(keys, t)) && clean_rows<DT, D, KT>(sv[t & 1], lane, wave)) odd = true;
    lds_barrier();  // the tile is there, and the one before it is done with
    if (t + 1 < tiles) load_k(t + 1), load_v(t + 1), load_bias(t + 1);
    scores(t);
    weights(t);
    values(t);
  }
  if (__syncthreads_or(odd)) {
#pragma unroll 1
    for (int t = 0; t < keys.tiles; ++t) {
      const int key = jag_key<KT>(keys, t);
      if (!in_part(key)) continue;
      load_v(t);
      brought();
      __syncthreads();
      mark_cols<DT, D, 4, false>(o, sv[t & 1], col_at, 0, [&](int j) { return sees(key + j); });
      __syncthreads();
    }
  }

  const float sum = l + __shfl_xor(l, 32);
  const int64_t at = (s.q0 + row) * a.hq + head;
  const float inv = sum != 0.0f ? 1.0f / sum : 0.0f;
  if (w0 < s.nq)
    store_own<DT, D, FINE>(o, inv, &sk[0][0] + wave * 32 * Tile<D>::RS, a.out, a.rest, ((s.q0 + w0) * a.hq + head) * D, (int64_t)a.hq * D, s.nq - w0);
  if (h == 0 && row < s.nq) {
    // log2 of the sum: of its mantissa, and its exponent beside the reference, whose rounding it shares
    if (a.lse)
      a.lse[at] = sum != 0.0f ? ((m + (float)__builtin_amdgcn_frexp_expf(sum)) + __builtin_amdgcn_logf(__builtin_amdgcn_frexp_mantf(sum))) * kLn2 : -kInf;
    if (a.stats) a.stats[2 * at] = sum != 0.0f ? m : kNoKeys, a.stats[2 * at + 1] = inv;
  }
  if constexpr (FINE) {
    const float far = l_far + __shfl_xor(l_far, 32), near = l_near + __shfl_xor(l_near, 32);
    float* outer = late_args().outer;
    if (outer && h == 0 && row < s.nq) outer[2 * at] = far * inv, outer[2 * at + 1] = near * inv;
  }
}

template <int DT, int D>
void launch(const JagArgs& a, hipStream_t st) {
  const int64_t units = a.items * a.hq, most = a.q_tokens > a.seqs ? a.q_tokens : a.seqs;
  const dim3 grid = linear_grid(units + (most + 255) / 256);
  if (a.bias) {
    if (a.rest) jag_fwd_kernel<DT, D, true, true><<<grid, 256, 0, st>>>(a, units);
    else jag_fwd_kernel<DT, D, true, false><<<grid, 256, 0, st>>>(a, units);
  } else {
    jag_fwd_kernel<DT, D, false, false><<<grid, 256, 0, st>>>(a, units);
  }
}

}  // namespace

int jag_args(const char* fn, const pdm_jagged_attention_desc* d, JagArgs& a) {
  auto bad = [&](const char* m) {
    set_error(std::string(fn) + ": " + m);
    return (int)PDM_ERR_INVALID;
  };
  if (!d) return bad("null descriptor");
  if (d->dtype != PDM_F16 && d->dtype != PDM_BF16) return bad("dtype must be F16 or BF16");
  if (d->head_dim != 64 && d->head_dim != 128) return bad("head_dim must be 64 or 128");
  if (d->n_kv_heads < 1 || d->n_q_heads < 1 || d->n_q_heads % d->n_kv_heads) return bad("n_q_heads must be a positive multiple of n_kv_heads");
  if (d->n_q_heads > 65535) return bad("at most 65535 query heads");
  if (d->num_seqs < 0 || d->num_seqs > (1 << 24)) return bad("num_seqs must lie in [0, 2^24]");
  if (d->q_tokens < 0 || d->k_tokens < 0 || d->q_tokens >= (1 << 30) || d->k_tokens >= (1 << 30)) return bad("tokens must lie in [0, 2^30)");
  if (d->q_tokens * d->n_q_heads >= (int64_t(1) << 31) || d->k_tokens * d->n_kv_heads >= (int64_t(1) << 31)) return bad("tokens * heads must be below 2^31");
  if (d->window < 0 || d->sinks < 0) return bad("window and sinks must not be negative");
  if (d->stats_planes < 0 || d->stats_planes > 2) return bad("stats_planes must lie in [0, 2]");
  const float scale2 = d->scale * kLog2e;
  if (!(scale2 - scale2 == 0.0f)) return bad("scale must be finite, and so must scale / ln 2");
  auto far = [](int64_t st) { return st < 0 || st >= (1 << 24); };
  if (far(d->q_stride_t) || far(d->k_stride_t) || far(d->v_stride_t)) return bad("token strides must lie in [0, 2^24)");
  if (d->bias_span < 0 || d->bias_span > (1 << 30)) return bad("bias_span must lie in [0, 2^30]");
  if (d->bias_start <= -(1 << 30) || d->bias_start >= (1 << 30)) return bad("bias_start must lie in (-2^30, 2^30)");
  a.seqs = d->num_seqs, a.hq = d->n_q_heads, a.hk = d->n_kv_heads, a.group = d->n_q_heads / d->n_kv_heads;
  a.q_tokens = d->q_tokens, a.k_tokens = d->k_tokens;
  a.causal = d->causal != 0;
  a.window = d->window >= d->k_tokens ? 0 : d->window;  // no distance reaches it
  a.sinks = a.window == 0 ? 0 : d->sinks < d->k_tokens ? d->sinks : (int32_t)d->k_tokens;
  a.bias_start = d->bias_start, a.bias_last = d->bias_span - 1;
  a.q_st = d->q_stride_t, a.q_sh = d->q_stride_h, a.k_st = d->k_stride_t, a.k_sh = d->k_stride_h;
  a.v_st = d->v_stride_t, a.v_sh = d->v_stride_h;
  a.scale = d->scale, a.scale2 = scale2;
  a.items = d->num_seqs ? d->q_tokens / 128 + d->num_seqs : 0;
  return PDM_OK;
}

int jag_inputs(const char* fn, JagArgs& a, const pdm_jagged_attention_desc* d, const void* q, const void* k, const void* v,
               const int32_t* cu_q, const int32_t* cu_k, const float* bias) {
  auto bad = [&](const char* m) {
    set_error(std::string(fn) + ": " + m);
    return (int)PDM_ERR_INVALID;
  };
  auto odd = [](const void* p, int64_t st, int64_t sh) { return (reinterpret_cast<uintptr_t>(p) & 15) || st % 8 || sh % 8; };
  if ((a.q_tokens && !q) || (a.k_tokens && (!k || !v))) return bad("null q / k / v");
  if (!cu_q || !cu_k) return bad("null cu_seqlens");
  if ((bias != nullptr) != (d->bias_span > 0)) return bad("bias and bias_span are given together");
  if (odd(q, a.q_st, a.q_sh) || odd(k, a.k_st, a.k_sh) || odd(v, a.v_st, a.v_sh))
    return bad("q, k and v must be 16-byte aligned, with strides that are multiples of 8");
  a.q = q, a.k = k, a.v = v, a.cu_q = cu_q, a.cu_k = cu_k, a.bias = bias;
  return PDM_OK;
}

}  // namespace pdm

using namespace pdm;

extern "C" int64_t pdm_jagged_attention_workspace_size(const pdm_jagged_attention_desc* desc) {
  clear_error();
  JagArgs a{};
  if (int e = jag_args(__func__, desc, a)) return e;
  return 0;
}

extern "C" int pdm_jagged_attention_fwd(const pdm_jagged_attention_desc* desc, const void* q, const void* k, const void* v,
                                        const int32_t* cu_q, const int32_t* cu_k, const float* bias, void* out, void* out_rest,
                                        float* lse, float* stats, void* workspace, int64_t workspace_bytes, int32_t* err_flag,
                                        pdm_stream_t stream) {
  clear_error();
  JagArgs a{};
  if (int e = jag_args(__func__, desc, a)) return e;
  if (a.q_tokens == 0 && (!err_flag || !a.seqs)) return PDM_OK;
  if (int e = jag_inputs(__func__, a, desc, q, k, v, cu_q, cu_k, bias)) return e;
  PDM_CHECK_ARG(out || !a.q_tokens, "null out");
  PDM_CHECK_ARG(!out_rest || bias, "out_rest without a bias");
  PDM_CHECK_ARG(((reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(out_rest)) & 15) == 0, "out and out_rest must be 16-byte aligned");
  PDM_CHECK_ARG(!out_rest || stats, "out_rest without stats");
  a.out = out, a.rest = out_rest, a.lse = lse, a.stats = stats, a.err = err_flag;
  if (out_rest && desc->stats_planes == 2) a.outer = stats + 2 * a.q_tokens * a.hq;
  const bool bf16 = desc->dtype == PDM_BF16;
  if (desc->head_dim == 64) bf16 ? launch<PDM_BF16, 64>(a, stream) : launch<PDM_F16, 64>(a, stream);
  else bf16 ? launch<PDM_BF16, 128>(a, stream) : launch<PDM_F16, 128>(a, stream);
  PDM_CHECK_LAUNCH();
  return PDM_OK;
}
