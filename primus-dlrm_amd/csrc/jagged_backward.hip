// Attention of ragged batches, backward, without atomics on memory: the same inputs give the same bits.
//
// With P the weights, dP = dO V^T and delta = rowsum(dO O) = rowsum(P dP):
//   dS = P (dP - delta),  dV = P^T dO,  dQ = scale dS K,  dK = scale dS^T Q,  dbias[c] = sum of dS over the pairs of column c.
// Two kernels compute S and dP again, one by blocks of queries (dQ, delta, the bias's gradient), one by blocks of keys (dK, dV):
// 7 products where one kernel would need 5 and sums of dQ over its workgroups, by atomics, whose order changes the result, or
// once more through memory in fp32.  In both a lane holds scores of one column (a query, a key) and passes them on to the next
// product as the first leaves them.
//
// P and dS are rounded to the type of the operands for their products; the bias's gradient takes dS in 32 bits.  fp16 would
// lose small dS (below 2^-14): its dS are multiplied by a power of two that brings the larger of dO and the gradient of lse to
// 2^-6, of each query for dQ, and of 32 queries for dK, whose sums so far are brought to it.  Weights for dV go in times 2^15, so
// that those down to 2^-29 keep all their bits; a larger dO would not bring them back.  (What is not finite does not count.
// dS of 2^20 times the largest |dO|, for which 64 values of 2^14 would have to point along dO, overflow.)
//
// Bound by latency at two waves a SIMD (matrix units 20 to 30 %, vector units 30 to 45, LDS 20 to 40 % of the time busy): 8
// sequences of 1,001 to 2,777 tokens, 8 heads of 64, both sides: 223 us by queries, of which the bias's gradient takes about
// half (sums of rows for its outer columns 12), and 196 by keys (0.55 PFLOP/s); 8,134 tokens, 24 heads of 128 on 6, window 512 with
// 4 sinks, fp16: 249, 230 and 46 for the sinks.
#include <algorithm>
#include <type_traits>

#include "jagged_common.h"

namespace pdm {

int jag_args(const char* fn, const pdm_jagged_attention_desc* d, JagArgs& a);
int jag_inputs(const char* fn, JagArgs& a, const pdm_jagged_attention_desc* d, const void* q, const void* k, const void* v,
               const int32_t* cu_q, const int32_t* cu_k, const float* bias);

namespace {

constexpr int M = 128;
constexpr int kOut = -5;     // |dO| and |dlse| below 2^kOut after their power of two
constexpr int kNone = -100;  // exponent of rows of zeros
constexpr float kLarge = 0x1p15f;  // fp16: weights, 1 at most, go into dV's product times this

// Rounded before the row's reference is taken off, which is a rounded score: the difference of the largest is 0, and not what rounding
// left of it, which from 2^30 on would count as 2^32 and more.
__device__ __forceinline__ float scaled(float score, float scale2) {
#pragma clang fp contract(off)
  return score * scale2;
}

__device__ __forceinline__ float sum16(const float* x) {  // four chains
  float s[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) s[i] = (x[i] + x[i + 4]) + (x[i + 8] + x[i + 12]);
  return (s[0] + s[1]) + (s[2] + s[3]);
}

__device__ __forceinline__ float pow2(int e) { return __builtin_amdgcn_ldexpf(1.0f, e); }

// ---- by queries -----------------------------------------------------------------------
// Gradients of the bias: sums along the diagonals of dS.  A wave writes 32 x 32 of them to LDS, row r shifted by 31 - r places in
// a line of 64 (the places that no row has stay zero), reads the lines back, a lane the sum of its place, and leaves its 63
// distances in a window.  (Atomic adds to LDS instead took 1,172 us for the sequences of 1,001 to 2,777 tokens below.)
// Distances fall from tile to tile; a thread sums those that are its number modulo 256 over the windows of the waves and writes
// each once, when the tiles have passed it.
template <int DT, int D, bool BIAS, bool GB>
__global__ void __launch_bounds__(256, 2) jag_dq_kernel(JagArgs a, int64_t units) {
  constexpr int KK = D / 16, DD = D / 32, KT = D == 64 ? 64 : 32, XX = KT / 32;  // (LDS for two workgroups on a CU)
  __shared__ alignas(1024) char sk[2][KT * Tile<D>::RS];
  __shared__ alignas(1024) char sv[2][KT * Tile<D>::RS];
  __shared__ float sb[2][BIAS ? M + KT : 1];
  __shared__ float win[2][GB ? 4 : 1][XX][GB ? 64 : 1];
  __shared__ alignas(1024) float lines[GB || D == 128 ? 4 : 1][GB || D == 128 ? 32 : 1][64];
  __shared__ float ends[GB ? 8 : 1];
  // Where registers are short three fragments of the queries stay in LDS: the compiler puts what does not fit into scratch memory,
  // whose load in every tile waits for the next tile's to land (fp16, 24 heads of 8,134 tokens under a window of 512: 256 us with
  // two, 240 with three).  bf16 still has one fragment there; a fourth would leave LDS for one workgroup on a CU.
  constexpr int HOLD = GB && D == 128 ? 3 : 0;
  __shared__ u32x4_t held[HOLD ? 4 * HOLD : 1][HOLD ? 64 : 1];
  __shared__ uint8_t odd_keys[2][KT];
  __shared__ int odd_any[2][4];

  const int64_t unit = linear_block();
  if (unit >= units) {
    const int64_t first = (unit - units) * 256;
    if (first >= a.q_tokens && first >= a.seqs) return;
    jag_guard(a, a.cu_q, a.q_tokens, first, [&](int64_t t) { clear_row(a.dq, t * a.hq * D, a.hq * D); });
    return;
  }
  const int hx = (int)(unit % a.hq), kh = hx % a.hk, head = kh * a.group + hx / a.hk;
  const int64_t place = unit / a.hq;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  JagSeq s;
  int b, r0;
  if (GB && hx == 0 && !jag_block<M>(a, a.cu_q, place, s, b, r0) && tid == 0)  // no partial result of that number
    a.part_range[2 * place] = 1, a.part_range[2 * place + 1] = 0;
  if (!(a.seqs <= 64 ? jag_ranked_block<M>(a, false, place, s, b, r0) : jag_block<M>(a, a.cu_q, a.items - 1 - place, s, b, r0))) return;
  const int64_t item = (s.q0 / M) + b + r0 / M;
  const int c = lane & 31, h = lane >> 5;
  const int off = s.nk - s.nq;
  const JagKeys keys = jag_keys<KT>(a, s, r0, (r0 + M < s.nq ? r0 + M : s.nq) - 1);

  const int row = r0 + wave * 32 + c, pos = off + row;
  const bool there = row < s.nq;
  struct Seen {  // keys that a query sees: [lo, lo + n) and those below first
    int lo, n, first;
    __device__ __forceinline__ bool operator()(int j) const { return (uint32_t)(j - lo) < (uint32_t)n || j < first; }
  };
  auto seen_from = [&](int p) {  // position p
    Seen x{0, 0, 0};
    if (p - off < s.nq) {
      const int hi = a.causal && p + 1 < s.nk ? (p + 1 > 0 ? p + 1 : 0) : s.nk;
      x.lo = a.window > 0 && p - a.window + 1 > 0 ? p - a.window + 1 : 0;
      x.n = hi > x.lo ? hi - x.lo : 0;
      x.first = a.sinks < hi ? a.sinks : hi;
    }
    return x;
  };
  const int64_t at = (s.q0 + row) * a.hq + head;
  // the wave's rows of q and dout, then of out and its rest, by way of the places of the tiles
  const int w0 = r0 + wave * 32, p_first = off + w0, p_last = off + (w0 + 31 < s.nq ? w0 + 31 : s.nq - 1);
  char *own = D == 64 ? &sk[0][0] + wave * 32 * Tile<D>::RS : (wave < 2 ? sk[wave & 1] : sv[wave & 1]);
  char *own2 = D == 64 ? &sv[0][0] + wave * 32 * Tile<D>::RS : reinterpret_cast<char*>(&lines[wave][0][0]);
  uint32_t row_at = Tile<D>::row_at(lane), col_at = Tile<D>::col_at(lane);
  const int64_t o_st = (int64_t)a.hq * D, o_at = s.q0 * o_st + head * D;
  u32x4_t q[KK], g[KK];
  float delta = 0.0f, most = 0.0f, m = 0.0f, inv = 0.0f;
  bring_own<D>(static_cast<const uint16_t*>(a.q) + s.q0 * a.q_st + head * a.q_sh, a.q_st, w0, s.nq, own);
  bring_own<D>(static_cast<const uint16_t*>(a.dout) + o_at, o_st, w0, s.nq, own2);
  brought();
#pragma unroll
  for (int kk = 0; kk < KK; ++kk) q[kk] = Tile<D>::rows(own, row_at, 0, kk), g[kk] = Tile<D>::rows(own2, row_at, 0, kk);
#pragma unroll
  for (int i = 0; i < HOLD; ++i) held[wave * HOLD + i][lane] = q[i];
  lds_barrier();
  bring_own<D>(static_cast<const uint16_t*>(a.out) + o_at, o_st, w0, s.nq, own);
  if (GB) bring_own<D>(static_cast<const uint16_t*>(a.rest) + o_at, o_st, w0, s.nq, own2);
  brought();
  // delta: the diagonal of the product of out's rows with dout's.  It is summed as dP is, of which it is a mean: where a row sees one
  // key, out is that key's value, and dS, the difference, is zero in all bits (a chain of additions left 1e-7 of |dO| |V|).
  constexpr f32x16_t zero16 = {0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
  f32x16_t od = zero16;
#pragma unroll
  for (int kk = 0; kk < KK; ++kk) od = mfma32<DT>(Tile<D>::rows(own, row_at, 0, kk), g[kk], od);
#pragma unroll
  for (int e = 0; e < 16; ++e) delta = c == 8 * (e >> 2) + 4 * h + (e & 3) ? od[e] : delta;
  const Seen mine_seen = seen_from(pos);
  const bool one_key = mine_seen.n + min(mine_seen.first, mine_seen.lo) == 1;
#pragma unroll
  for (int kk = 0; kk < KK; ++kk) {
    u32x4_t o = {0, 0, 0, 0}, o2 = {0, 0, 0, 0};
    if (GB) o = Tile<D>::rows(own, row_at, 0, kk), o2 = Tile<D>::rows(own2, row_at, 0, kk);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float lo = lo_of<DT>(g[kk][e]), hi = hi_of<DT>(g[kk][e]);
      if (GB && !one_key) {
        delta = __builtin_fmaf(lo, rest_lo<DT>(o[e], o2[e]), delta);
        delta = __builtin_fmaf(hi, rest_hi<DT>(o[e], o2[e]), delta);
      }
      if (DT == PDM_F16) most = fmaxf(most, fmaxf(fabsf(lo) < kInf ? fabsf(lo) : 0.0f, fabsf(hi) < kInf ? fabsf(hi) : 0.0f));
    }
  }
  delta += __shfl_xor(delta, 32);
  lds_barrier();
  if (there && a.dlse) {  // d lse / d s = P
    const float x = a.dlse[at];
    delta -= x;
    if (DT == PDM_F16 && fabsf(x) < kInf) most = fmaxf(most, fabsf(x));
  }
  float back = a.scale, ahead = 1.0f;  // fp16: the row's power of two
  if (DT == PDM_F16) {
    most = fmaxf(most, __shfl_xor(most, 32));
    const int e = most > 0.0f ? __builtin_amdgcn_frexp_expf(most) : kNone;
    const int of = (int)group_max((float)e, 64);
    if (lane == 0 && r0 + wave * 32 < s.nq) a.expo[(item * 4 + wave) * a.hq + head] = of;
    if (e != kNone) ahead = pow2(kOut - e), back = a.scale * pow2(e - kOut);
  }
  if (there) {
    m = a.stats[2 * at], inv = a.stats[2 * at + 1];
    if (h == 0) a.delta[at] = delta;
  }

  const uint16_t* kp = static_cast<const uint16_t*>(a.k) + s.k0 * a.k_st + kh * a.k_sh;
  const uint16_t* vp = static_cast<const uint16_t*>(a.v) + s.k0 * a.v_st + kh * a.v_sh;
  const float* brow = BIAS ? a.bias + (int64_t)head * (a.bias_last + 1) : nullptr;
  Bring<D, KT> bring_k, bring_v;
  bring_k.init(a.k_st, lane, wave);
  bring_v.init(a.v_st, lane, wave);
  float bias_next = 0.0f;
  const int bias_at = bias_from(a, (int64_t)off + r0 - (KT - 1));
  auto load = [&](int t) {
    const int key = jag_key<KT>(keys, t);
    bring_k.load(kp, a.k_st, key, s.nk, sk[t & 1], wave);
    bring_v.load(vp, a.v_st, key, s.nk, sv[t & 1], wave);
    if (BIAS && tid < M + KT) bias_next = bias2(a, brow, bias_at - key + tid);
  };

  // the bias's gradient: columns 0 .. cols - 1 of the partial result, then what lies behind them and before them
  const int cols = (int)a.part_stride - 2;
  float* part = GB ? a.part + (item * a.hq + head) * a.part_stride : nullptr;
  float far = 0.0f, near = 0.0f, all = 0.0f, sum = 0.0f;  // all: of this row's dS
  int mine = 0;  // the distance that this thread sums
  auto put = [&](int d, float v) {
    const int x = d - a.bias_start;
    if (x >= 0 && x < cols) part[x] = v;
  };
  auto gather = [&](int t) {  // the windows of tile t
    const int base = off + r0 - jag_key<KT>(keys, t) - (KT - 1), rel = (tid - base) & 255;
    if (t == 0) {
      mine = base + rel;
    } else if (mine != base + rel) {
      put(mine, sum);
      mine -= 256;
      const int over = mine - (a.bias_start + cols - 1);  // distances of no column: passed at once
      if (over > 0) mine -= min(mine - base - rel, (over + 255) & ~255);
      for (; mine > base + rel; mine -= 256) put(mine, 0.0f);
      sum = 0.0f;
    }
#pragma unroll
    for (int w = 0; w < 4; ++w) {
#pragma unroll
      for (int x = 0; x < XX; ++x) {
        const int place = rel - 32 * w - 32 * (XX - 1 - x);
        if (place >= 0 && place < 63) sum += win[t & 1][w][x][place];
      }
    }
  };
  if (GB) {
    float* w = &lines[0][0][0];
    for (int i = tid; i < 4 * 32 * 64; i += 256) w[i] = 0.0f;
    if (hx == 0 && tid == 0) {
      a.part_range[2 * item] = keys.tiles ? off + r0 - jag_key<KT>(keys, keys.tiles - 1) - (KT - 1) : 1;
      a.part_range[2 * item + 1] = keys.tiles ? off + r0 - jag_key<KT>(keys, 0) + M - 1 : 0;
    }
  }

  f32x16_t dq[DD];
#pragma unroll
  for (int d = 0; d < DD; ++d) dq[d] = zero16;

  auto unseen = [&](int key) {  // (as in the forward pass)
    return w0 >= s.nq || (a.causal && key > p_last) || (a.window > 0 && key + KT - 1 <= p_first - a.window && key >= a.sinks);
  };
  auto all_seen = [&](int key) {
    return key + KT <= s.nk && (!a.causal || key + KT - 1 <= p_first) && (a.window == 0 || key > p_last - a.window || key + KT <= a.sinks);
  };
  const int b_first = off + r0, b_last = off + (r0 + M < s.nq ? r0 + M : s.nq) - 1;
  auto in_part = [&](int key) {
    return (a.causal && key + KT - 1 > b_first) || (a.window > 0 && key <= b_last - a.window && key + KT > a.sinks);
  };
  bool odd = false;
  if (keys.tiles > 0) load(0);
#pragma unroll 1
  for (int t = 0; t < keys.tiles; ++t) {
    const int key = jag_key<KT>(keys, t);
    if (BIAS && tid < M + KT) sb[t & 1][tid] = bias_next;
    brought();
    const bool part_seen = in_part(key);
    if (part_seen) {
      const bool bad = clean_rows<DT, D, KT>(sk[t & 1], lane, wave, odd_keys[t & 1]);
      odd = odd || bad;
      if (lane == 0) odd_any[t & 1][wave] = bad;
    }
    lds_barrier();  // the tile is there, and the one before it is done with
    if (t + 1 < keys.tiles) load(t + 1);
    if (GB && t > 0) gather(t - 1);
    if (unseen(key)) {
#pragma unroll
      for (int x = 0; x < XX; ++x)
        if (GB) win[t & 1][wave][x][lane] = 0.0f;
      continue;
    }
    const char *tk = sk[t & 1], *tv = sv[t & 1];
    const bool whole = all_seen(key);
#pragma unroll
    for (int x = 0; x < XX; ++x) {
      if (D == 128) asm volatile("" : "+v"(row_at), "+v"(col_at));  // places are computed here, not held through the loop
      f32x16_t sc = zero16, dp = zero16;
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) {
        sc = mfma32<DT>(Tile<D>::rows(tk, row_at, 32 * x, kk), kk < HOLD ? held[wave * HOLD + kk][lane] : q[kk], sc);
        dp = mfma32<DT>(Tile<D>::rows(tv, row_at, 32 * x, kk), g[kk], dp);
      }
      sched_mfma_ds_pipeline<2 * KK, 4>();
      __builtin_amdgcn_sched_barrier(0);
      float ds[16];
      const int local = c - 32 * x - 4 * h + KT - 1;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int j = 8 * (e >> 2) + (e & 3);
        const float w = BIAS ? __builtin_fmaf(sc[e], a.scale2, sb[t & 1][wave * 32 + local - j]) - m : scaled(sc[e], a.scale2) - m;
        const float p = __builtin_amdgcn_exp2f(w) * inv;
        ds[e] = p * (dp[e] - delta);
      }
      if (part_seen && (odd_any[t & 1][0] | odd_any[t & 1][1] | odd_any[t & 1][2] | odd_any[t & 1][3])) {
        // a key that is not finite: scores of -inf, or rows of NaN
#pragma unroll 1
        for (int w = 0; w < 4; ++w) {
          if (!odd_any[t & 1][w]) continue;
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const int j = 32 * x + 4 * h + 8 * (e >> 2) + (e & 3);
            if (j / (KT / 4) == w && odd_keys[t & 1][j] && inv == inv) ds[e] = 0.0f;
          }
        }
      }
      if (!whole) {
        int p = pos;
        if (D == 128) asm volatile("" : "+v"(p));  // not held through the loop
        const Seen sees = seen_from(p);
#pragma unroll
        for (int e = 0; e < 16; ++e) ds[e] = sees(key + 32 * x + 4 * h + 8 * (e >> 2) + (e & 3)) ? ds[e] : 0.0f;
      }
      if (GB) all += sum16(ds);
      bool near_lines = false;
      if (GB) {
        const int first = p_first - key - 32 * x - 31 - a.bias_start, last = first + 62;  // columns of the wave's pairs
        const int col = pos - key - 32 * x - 4 * h - a.bias_start;
        near_lines = first < a.bias_last && last >= 0;
        // Rows that are not there stay out of these sums (their places in the lines stay zero): nothing holds their weights, which
        // are the bias's alone, and infinity times 0 for a large one.
        if (there) {
          if (first >= a.bias_last) {
            far += sum16(ds);
          } else if (last < 0) {
            near += sum16(ds);
          } else {
            float* line = &lines[wave][4 * h][c + 31 - 4 * h];
            if (first >= 0 && last < a.bias_last) {
#pragma unroll
              for (int e = 0; e < 16; ++e) line[(8 * (e >> 2) + (e & 3)) * 63] = ds[e];
            } else {
#pragma unroll
              for (int e = 0; e < 16; ++e) {
                const int j = 8 * (e >> 2) + (e & 3), y = col - j;
                far += y >= a.bias_last ? ds[e] : 0.0f;
                near += y < 0 ? ds[e] : 0.0f;
                line[j * 63] = y >= 0 && y < a.bias_last ? ds[e] : 0.0f;
              }
            }
          }
        }
      }
      u32x4_t w[2];
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e >> 2][e & 3] = DT == PDM_F16 ? pack2<DT>(ds[2 * e] * ahead, ds[2 * e + 1] * ahead) : pack2<DT>(ds[2 * e], ds[2 * e + 1]);
      add_cols<DT, D, 2>(dq, tk, col_at, 32 * x, w);
      if (GB) {
        float along = 0.0f;
        if (near_lines) {
          own_lds_order();
#pragma unroll
          for (int r = 0; r < 32; r += 4)
            along += (lines[wave][r][lane] + lines[wave][r + 1][lane]) + (lines[wave][r + 2][lane] + lines[wave][r + 3][lane]);
          own_lds_order();
        }
        win[t & 1][wave][x][lane] = along;
      }
    }
  }
  if (GB) {
    __syncthreads();
    if (keys.tiles > 0) {
      gather(keys.tiles - 1);
      put(mine, sum);
    }
    // A row's dS add up to the gradient of its lse.  What they are off by is delta's error, which each has by its weight: little beside
    // its own size, but a column of nearly all weights of every row has a sum that cancels to far less than its terms.  So the two
    // columns that stand for many distances are put right (a bias of two columns, 980 tokens, and this and what rest2 keeps left
    // out: off by 1.2e-5 to 8.6e-5 of the gradient, with both by 9e-7 to 2.8e-6).
    // A bias of one column has all of a row, whose sum is known.
    const float sum_of_row = all + __shfl_xor(all, 32);
    const JagArgs& late = late_args();
    if (late.outer && there && fabsf(sum_of_row) < kInf) {
      const float right = late.dlse ? late.dlse[at] : 0.0f, p_far = late.outer[2 * at], p_near = late.outer[2 * at + 1];
      if (a.bias_last == 0) far = h == 0 && p_far + p_near > 0.5f ? right : 0.0f, near = 0.0f;
      else if (h == 0) far -= (sum_of_row - right) * p_far, near -= (sum_of_row - right) * p_near;
    }
    far = group_sum(far, 64), near = group_sum(near, 64);
    if (lane == 0) ends[wave] = far, ends[4 + wave] = near;
    __syncthreads();
    if (tid < 2) part[cols + tid] = (ends[4 * tid] + ends[4 * tid + 1]) + (ends[4 * tid + 2] + ends[4 * tid + 3]);
  }
  if (__syncthreads_or(odd)) {
    const Seen sees = seen_from(pos);
#pragma unroll 1
    for (int t = 0; t < keys.tiles; ++t) {
      const int key = jag_key<KT>(keys, t);
      if (!in_part(key)) continue;
      load(t);
      brought();
      __syncthreads();
      mark_cols<DT, D, 2 * XX, true>(dq, sk[t & 1], col_at, 0, [&](int j) { return sees(key + j); });
      __syncthreads();
    }
  }
  if (w0 < s.nq)
    store_own<DT, D>(dq, back, D == 64 ? own : own2, late_args().dq, nullptr, o_at + w0 * o_st, o_st, s.nq - w0);
}

// Sums the partial gradients of a column over the blocks of queries, in 64 bits: a lane per column, the blocks dealt to 16 waves.
__global__ void __launch_bounds__(1024) jag_dbias_kernel(JagArgs a) {
  __shared__ double part[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, cols = (int)a.part_stride - 2;
  const int head = blockIdx.y, col = (int)(blockIdx.z * gridDim.x + blockIdx.x) * 64 + lane;
  double sum = 0.0;
  const int64_t d = (int64_t)col + a.bias_start;
  for (int64_t i0 = wave; i0 < a.items; i0 += 16 * 64) {  // 64 blocks' ranges at once, a lane's each
    const int64_t mine = i0 + 16 * lane;
    int lo = 1, hi = 0;
    if (mine < a.items) lo = a.part_range[2 * mine], hi = a.part_range[2 * mine + 1];
    const int n = a.items - i0 < 16 * 64 ? (int)((a.items - i0 + 15) / 16) : 64;
#pragma unroll 4
    for (int j = 0; j < n; ++j) {
      const int from = __builtin_amdgcn_readlane(lo, j), to = __builtin_amdgcn_readlane(hi, j);
      const float* p = a.part + ((i0 + 16 * j) * a.hq + head) * a.part_stride;
      float v = 0.0f;
      if (from <= to) {
        if (col < cols && col < a.bias_last && d >= from && d <= to) v = p[col];
        if (col == a.bias_last) v = p[cols];
        if (col == 0) v += p[cols + 1];
      }
      sum += v;
    }
  }
  part[wave][lane] = sum;
  __syncthreads();
  if (wave || col > a.bias_last) return;
  for (int w = 1; w < 16; ++w) sum += part[w][lane];
  a.dbias[(int64_t)head * (a.bias_last + 1) + col] = (float)sum;
}

// ---- by keys ----------------------------------------------------------------------------
// A workgroup takes 128 keys of a key head, 32 a wave, and walks the queries that see them under the window, head by head of the
// group.  Sums of 128 elements take half of the registers of two waves, so there K is read from LDS for every product.
//
// First tokens that stay visible (SINK) have many more queries than other keys: those beyond the window are a kernel of their
// own, a workgroup per 32 such keys and a share of these queries, which its waves take in turn.  Both leave sums in fp32, which
// jag_sinks_kernel joins and rounds.
//
// Only a sequence longer than the window has such queries, and only for its first nk - window keys.  The host does not know the
// lengths: blocks are listed (sink_list), and have rows for their sums (sink_cell), by sequence (0), or by cells of window + 1 keys of
// the batch, either where it is less.  A sequence of nk > window keys from k0 on has the nk / (window + 1) cells from number
// k0 / (window + 1) on to itself, and its sums fit into min(sinks, window + 1) rows of each.  (1,000 sequences of 100 tokens, a window
// of 1 with 200 sinks, listed by cells: the pass took 4,970 us instead of 3,058.  16,384 sequences of 100 tokens, 8 key heads of 128, a
// window of 1,024 with 4 sinks: 0.1 GB and not 8.6.)
__device__ __forceinline__ int sinks_with_far_queries(const JagArgs& a, const JagSeq& s) {
  return a.sink_blocks ? max(0, min(a.sinks, s.nk - a.window)) : 0;
}

// Block x of the list: keys [j0, j0 + n) of sequence b, n <= 32.  False for one without keys.
__device__ __forceinline__ bool sink_block(const JagArgs& a, int64_t x, JagSeq& s, int& b, int& j0, int& n) {
  int64_t block = x % a.sink_blocks;
  x /= a.sink_blocks;
  b = a.sink_list ? find_sequence(a.seqs, (x + 1) * a.sink_list - 1, [&](int i) { return (int64_t)a.cu_k[i]; }) : (int)x;
  if (!jag_seq(a, b, s)) return false;
  if (a.sink_list) block += (x - s.k0 / a.sink_list) * a.sink_blocks;
  const int rows = sinks_with_far_queries(a, s);
  if (block < 0 || block * 32 >= rows) return false;
  j0 = (int)block * 32, n = min(32, rows - j0);
  return true;
}

// The sums of such a block and key head: [shares + 1][dk, dv][D][n], the last for the queries under the window.
template <int D>
__device__ __forceinline__ float* sink_sums(const JagArgs& a, const JagSeq& s, int b, int j0, int n, int kh) {
  const int64_t row = (a.sink_cell ? s.k0 / a.sink_cell : b) * a.sink_rows + j0;
  return a.sink_part + (row * a.hk + kh * n) * (a.sink_shares + 1) * (2 * D);
}

template <int DT, int D, bool BIAS, bool SINK>
__global__ void __launch_bounds__(256, SINK ? 1 : 2) jag_dkv_kernel(JagArgs a, int64_t units) {
  constexpr int KK = D / 16, DD = D / 32;
  constexpr int QT = SINK ? 128 : D == 64 ? 64 : 32, KEYS = SINK ? 32 : M;
  constexpr bool KL = D == 128 && !SINK;   // K in LDS
  __shared__ alignas(1024) char sq[2][QT * Tile<D>::RS];
  __shared__ alignas(1024) char sg[2][QT * Tile<D>::RS];
  __shared__ alignas(1024) char sk[KL ? KEYS * Tile<D>::RS : 16];
  __shared__ float sb[2][BIAS ? KEYS + QT : 1];
  __shared__ alignas(16) float ss[2][3 * QT + 4];  // of the tile's queries: reference, 1 / sum, delta; fp16: the exponents of each 32
  constexpr int STATS = 3 * QT + (DT == PDM_F16 ? QT / 32 : 0);

  const int64_t unit = linear_block();
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 31, h = lane >> 5;
  JagSeq s;
  int b, j0, kh, share = 0, keys_n = 0;  // SINK: its share of the queries, its keys
  if constexpr (SINK) {
    if (unit >= units) return;
    share = (int)(unit % a.sink_shares);
    const int64_t x = unit / a.sink_shares;
    kh = (int)(x % a.hk);
    if (!sink_block(a, x / a.hk, s, b, j0, keys_n)) return;
  } else {
    if (unit >= units) {
      const int64_t first = (unit - units) * 256;
      if (first >= a.k_tokens && first >= a.seqs) return;
      jag_guard(a, a.cu_k, a.k_tokens, first, [&](int64_t t) {
        clear_row(a.dk, t * a.hk * D, a.hk * D);
        clear_row(a.dv, t * a.hk * D, a.hk * D);
      });
      return;
    }
    kh = (int)(unit % a.hk);
    if (!(a.seqs <= 64 ? jag_ranked_block<M>(a, true, unit / a.hk, s, b, j0) : jag_block<M>(a, a.cu_k, unit / a.hk, s, b, j0))) return;
  }
  const int off = s.nk - s.nq, jw = SINK ? j0 : j0 + wave * 32;
  // queries that see a key of the block
  const int j1 = (j0 + KEYS < s.nk ? j0 + KEYS : s.nk) - 1;
  int i_lo = a.causal && j0 - off > 0 ? j0 - off : 0, i_hi = s.nq;
  if (SINK) i_lo = j0 + a.window - off > 0 ? j0 + a.window - off : 0;
  else if (a.window > 0 && j1 + a.window - off < i_hi) i_hi = j1 + a.window - off;
  i_lo &= ~(QT - 1);
  const int tiles = i_hi > i_lo ? (i_hi - i_lo + QT - 1) / QT : 0;
  const int64_t all = (int64_t)tiles * a.group;
  const int n0 = SINK ? (int)(all * share / a.sink_shares) : 0, n1 = SINK ? (int)(all * (share + 1) / a.sink_shares) : (int)all;

  // this lane's key and the queries that see it here: [see_lo, see_lo + see_n)
  const int key = jw + c;
  const bool there = key < s.nk;
  int see_lo = 0, see_n = 0;
  if (there && !(SINK && key >= a.sinks)) {
    const int edge = key + a.window - off;
    see_lo = SINK ? (edge > 0 ? edge : 0) : a.causal && key - off > 0 ? key - off : 0;
    const int hi = !SINK && a.window > 0 && edge < s.nq ? edge : s.nq;
    see_n = hi > see_lo ? hi - see_lo : 0;
  }
  uint32_t row_at = Tile<D>::row_at(lane), col_at = Tile<D>::col_at(lane);
  // the wave's keys and values, by way of the places of the tiles
  const int64_t k_at = s.k0 * a.k_st + kh * a.k_sh, v_at = s.k0 * a.v_st + kh * a.v_sh;
  char* own = SINK || D == 64 ? &sq[0][0] + wave * 32 * Tile<D>::RS : (wave < 2 ? sq[wave & 1] : sg[wave & 1]);
  u32x4_t kf[KL ? 1 : KK], vf[KK];
  if constexpr (KL) {
    bring_own<D>(static_cast<const uint16_t*>(a.v) + v_at, a.v_st, jw, s.nk, own);
    Bring<D, KEYS> bring_k;
    bring_k.init(a.k_st, lane, wave);
    bring_k.load(static_cast<const uint16_t*>(a.k) + k_at, a.k_st, j0, s.nk, sk, wave);
    brought();
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) vf[kk] = Tile<D>::rows(own, row_at, 0, kk);
    lds_barrier();
  } else {
    char* own2 = &sg[0][0] + wave * 32 * Tile<D>::RS;
    bring_own<D>(static_cast<const uint16_t*>(a.v) + v_at, a.v_st, jw, s.nk, own);
    bring_own<D>(static_cast<const uint16_t*>(a.k) + k_at, a.k_st, jw, s.nk, own2);
    brought();
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) vf[kk] = Tile<D>::rows(own, row_at, 0, kk), kf[kk] = Tile<D>::rows(own2, row_at, 0, kk);
    lds_barrier();
  }

  Bring<D, QT> bring_q, bring_g;
  const int64_t g_st = (int64_t)a.hq * D, item0 = s.q0 / M + b;
  bring_q.init(a.q_st, lane, wave);
  bring_g.init(g_st, lane, wave);
  float bias_next = 0.0f, stat_next[QT == 128 ? 2 : 1];
  int head_next = tiles ? n0 / tiles : 0, tile_next = tiles ? n0 % tiles : 0;
  // (No load from memory may stand between these and their use: it would wait for them.  The exponents, read where they were needed,
  // cost 236 us instead of 227.)
  auto load = [&](int n) {  // the head and tile at which the next load stands
    const int head = kh * a.group + head_next, i = i_lo + tile_next * QT;
    bring_q.load(static_cast<const uint16_t*>(a.q) + s.q0 * a.q_st + head * a.q_sh, a.q_st, i, s.nq, sq[n & 1], wave);
    bring_g.load(static_cast<const uint16_t*>(a.dout) + s.q0 * g_st + head * D, g_st, i, s.nq, sg[n & 1], wave);
    if (BIAS && tid < KEYS + QT) bias_next = bias2(a, a.bias + (int64_t)head * (a.bias_last + 1), bias_from(a, (int64_t)off + i - (KEYS - 1) - j0) + tid);
#pragma unroll
    for (int u = 0; u < (QT == 128 ? 2 : 1); ++u) {
      const int x = tid + 256 * u, r = i + (x & (QT - 1)), g = i + 32 * (x - 3 * QT);
      stat_next[u] = 0.0f;
      if (x < 3 * QT && r < s.nq) {
        const int64_t at = (s.q0 + r) * a.hq + head;
        stat_next[u] = x < QT ? a.stats[2 * at] : x < 2 * QT ? a.stats[2 * at + 1] : a.delta[at];
      }
      if (x >= 3 * QT && x < STATS && g < s.nq) stat_next[u] = __int_as_float(a.expo[((item0 + (g >> 7)) * 4 + (g >> 5 & 3)) * a.hq + head]);
    }
    if (++tile_next == tiles) tile_next = 0, ++head_next;
  };

  constexpr f32x16_t zero16 = {0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
  f32x16_t dk[DD], dv[DD];
#pragma unroll
  for (int d = 0; d < DD; ++d) dk[d] = zero16, dv[d] = zero16;
  int power = 100;  // fp16: dk holds sums times 2^power

  // of 32 queries: none sees a key of this wave; each sees all of them (here); of a query: it sees this lane's key
  auto unseen = [&](int i) {
    const int p0 = off + i;
    return i >= s.nq || jw >= s.nk || (SINK ? p0 + 31 < jw + a.window : (a.causal && p0 + 31 < jw) || (a.window > 0 && p0 >= jw + 31 + a.window));
  };
  auto all_seen = [&](int i) {
    const int p0 = off + i;
    return i + 32 <= s.nq && jw + 32 <= (SINK && a.sinks < s.nk ? a.sinks : s.nk) &&
           (SINK ? p0 >= jw + 31 + a.window : (!a.causal || p0 >= jw + 31) && (a.window == 0 || p0 + 31 < jw + a.window));
  };
  // some pair of the tile's queries and the workgroup's keys is not seen (what lies behind the last query comes as zeros)
  auto in_part = [&](int i) {
    const int p0 = off + i;
    if (SINK) return p0 < j1 + a.window || j1 >= a.sinks;
    return (a.causal && p0 < j1) || (a.window > 0 && p0 + QT - 1 >= j0 + a.window);
  };
  auto sees = [&](int i) { return (uint32_t)(i - see_lo) < (uint32_t)see_n; };
  bool odd = false;
  int tt = tile_next;
  if (n1 > n0) load(n0);
#pragma unroll 1
  for (int n = n0; n < n1; ++n) {
    const int i0 = i_lo + tt * QT;
    if (++tt == tiles) tt = 0;
    if (BIAS && tid < KEYS + QT) sb[n & 1][tid] = bias_next;
#pragma unroll
    for (int u = 0; u < (QT == 128 ? 2 : 1); ++u)
      if (const int x = tid + 256 * u; x < STATS) ss[n & 1][x] = DT == PDM_F16 && x >= QT && x < 2 * QT ? stat_next[u] * kLarge : stat_next[u];
    brought();
    if (in_part(i0)) {
      if (clean_rows<DT, D, QT>(sq[n & 1], lane, wave)) odd = true;
      if (clean_rows<DT, D, QT>(sg[n & 1], lane, wave)) odd = true;
    }
    lds_barrier();  // the tile is there, and the one before it is done with
    if (n + 1 < n1) load(n + 1);
    const char *tq = sq[n & 1], *tg = sg[n & 1];
#pragma unroll
    for (int y0 = 0; y0 < (SINK ? 1 : QT / 32); ++y0) {
      const int x = SINK ? wave : y0, i = i0 + 32 * x;
      if (unseen(i)) continue;
      const bool whole = all_seen(i);
      if (D == 128) asm volatile("" : "+v"(row_at), "+v"(col_at));  // places are computed here, not held through the loop
      f32x16_t sc = zero16, dp = zero16;
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) {
        u32x4_t f;
        if constexpr (KL) f = Tile<D>::rows(sk, row_at, 32 * wave, kk);
        else f = kf[kk];
        sc = mfma32<DT>(Tile<D>::rows(tq, row_at, 32 * x, kk), f, sc);
        dp = mfma32<DT>(Tile<D>::rows(tg, row_at, 32 * x, kk), vf[kk], dp);
      }
      if constexpr (!KL) sched_mfma_ds_pipeline<2 * KK, 4>();
      __builtin_amdgcn_sched_barrier(0);
      float ahead = 1.0f;
      if (DT == PDM_F16) {
        const int want = kOut - __builtin_amdgcn_readfirstlane(__float_as_int(ss[n & 1][3 * QT + x]));
        if (want < power) {  // larger gradients than any before
          const float f = pow2(want - power);
          power = want;
#pragma unroll
          for (int d = 0; d < DD; ++d) dk[d] *= f;
        }
        ahead = pow2(power) / kLarge;
      }
      float p[16], ds[16];  // fp16: times kLarge
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        const int r = 32 * x + 8 * y + 4 * h;
        const f32x4_t m = *reinterpret_cast<const f32x4_t*>(&ss[n & 1][r]), inv = *reinterpret_cast<const f32x4_t*>(&ss[n & 1][QT + r]);
        const f32x4_t delta = *reinterpret_cast<const f32x4_t*>(&ss[n & 1][2 * QT + r]);
#pragma unroll
        for (int z = 0; z < 4; ++z) {
          const int e = 4 * y + z;
          const float w = BIAS ? __builtin_fmaf(sc[e], a.scale2, sb[n & 1][r + z - (jw - j0) - c + KEYS - 1]) - m[z] : scaled(sc[e], a.scale2) - m[z];
          p[e] = __builtin_amdgcn_exp2f(w) * inv[z];
          ds[e] = p[e] * (dp[e] - delta[z]);
        }
      }
      if (!whole) {
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const bool ok = sees(i + 4 * h + 8 * (e >> 2) + (e & 3));
          p[e] = ok ? p[e] : 0.0f, ds[e] = ok ? ds[e] : 0.0f;
        }
      }
      u32x4_t pw[2], dw[2];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        pw[e >> 2][e & 3] = pack2<DT>(p[2 * e], p[2 * e + 1]);
        dw[e >> 2][e & 3] = DT == PDM_F16 ? pack2<DT>(ds[2 * e] * ahead, ds[2 * e + 1] * ahead) : pack2<DT>(ds[2 * e], ds[2 * e + 1]);
      }
      add_cols<DT, D, 2>(dv, tg, col_at, 32 * x, pw);
      add_cols<DT, D, 2>(dk, tq, col_at, 32 * x, dw);
    }
  }
  if (__syncthreads_or(odd)) {
    head_next = tiles ? n0 / tiles : 0, tile_next = tiles ? n0 % tiles : 0;
#pragma unroll 1
    for (int n = n0; n < n1; ++n) {
      const int i0 = i_lo + tile_next * QT;
      load(n);
      brought();
      __syncthreads();
#pragma unroll 1
      for (int y0 = 0; y0 < (SINK ? 1 : QT / 32); ++y0) {
        const int x = SINK ? wave : y0;
        if (!in_part(i0)) continue;
        mark_cols<DT, D, 2, false>(dv, sg[n & 1], col_at, 32 * x, [&](int r) { return sees(i0 + r); });
        mark_cols<DT, D, 2, true>(dk, sq[n & 1], col_at, 32 * x, [&](int r) { return sees(i0 + r); });
      }
      __syncthreads();
    }
  }
  const JagArgs& late = late_args();
  const float back = DT == PDM_F16 ? pow2(-power) : 1.0f, back_v = DT == PDM_F16 ? 1.0f / kLarge : 1.0f;
  if constexpr (SINK) {
    float* to = sink_sums<D>(late, s, b, j0, keys_n, kh) + (int64_t)share * (2 * D) * keys_n;
    float* mine = reinterpret_cast<float*>(wave < 2 ? sq[wave & 1] : sg[wave & 1]);  // QT rows of a tile: D x 32 floats and more
#pragma unroll
    for (int z = 0; z < 2; ++z) {
      __syncthreads();  // the tiles, or the sums before, are done with
#pragma unroll
      for (int d = 0; d < DD; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) mine[(32 * d + 8 * (e >> 2) + 4 * h + (e & 3)) * 32 + c] = z ? dv[d][e] * back_v : dk[d][e] * back;
      __syncthreads();
      for (int i = tid; i < D * keys_n; i += 256) {
        const int d = i / keys_n, x = 32 * d + (i - d * keys_n);
        to[z * D * keys_n + i] = (reinterpret_cast<const float*>(sq[0])[x] + reinterpret_cast<const float*>(sq[1])[x]) +
                                 (reinterpret_cast<const float*>(sg[0])[x] + reinterpret_cast<const float*>(sg[1])[x]);
      }
    }
    return;
  }
  const int n = min(32, sinks_with_far_queries(late, s) - jw);
  if (c < n) {  // jag_sinks_kernel writes over what these rows get below
    float* to = sink_sums<D>(late, s, b, jw, n, kh) + (int64_t)late.sink_shares * (2 * D) * n;
#pragma unroll
    for (int d = 0; d < DD; ++d)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int x = (32 * d + 8 * (e >> 2) + 4 * h + (e & 3)) * n + c;
        to[x] = dk[d][e] * back, to[D * n + x] = dv[d][e] * back_v;
      }
  }
  if (jw >= s.nk) return;
  const int64_t at = ((s.k0 + jw) * late.hk + kh) * D, st = (int64_t)late.hk * D;
  store_own<DT, D>(dk, late.scale * back, own, late.dk, nullptr, at, st, s.nk - jw);
  store_own<DT, D>(dv, back_v, own, late.dv, nullptr, at, st, s.nk - jw);
}

// Gradients of a block of sinks of a key head, their sums under the window and beyond it: a thread an element at a time, `parts`
// workgroups.
template <int DT, int D>
__global__ void __launch_bounds__(256) jag_sinks_kernel(JagArgs a, int64_t units, int parts) {
  const int64_t unit = linear_block() / parts;
  if (unit >= units) return;
  const int kh = (int)(unit % a.hk);
  JagSeq s;
  int b, j0, n;
  if (!sink_block(a, unit / a.hk, s, b, j0, n)) return;
  const float* from = sink_sums<D>(a, s, b, j0, n, kh);
  for (int i = (int)(linear_block() % parts) * 256 + threadIdx.x; i < 2 * D * n; i += parts * 256) {
    const int z = i / (D * n), d = i / n % D, key = j0 + i % n;
    float sum = 0.0f;
#pragma unroll 4
    for (int x = 0; x <= a.sink_shares; ++x) sum += from[(int64_t)x * (2 * D) * n + i];
    static_cast<uint16_t*>(z ? a.dv : a.dk)[((s.k0 + key) * a.hk + kh) * D + d] = (uint16_t)pack2<DT>(z ? sum : sum * a.scale, 0.0f);
  }
}

// ---- host -------------------------------------------------------------------------------
int64_t round256(int64_t v) { return (v + 255) / 256 * 256; }

// Columns of a partial gradient of the bias: those that a distance of the batch may reach, but for the last.
int64_t part_cols(const JagArgs& a) {
  const int64_t reach = a.k_tokens - a.bias_start;
  return reach < 0 ? 0 : reach < a.bias_last ? reach : a.bias_last;
}

// The list of blocks of 32 sinks (jag_dkv_kernel), and the shares that the queries beyond the window are dealt to: about 1,024
// workgroups, each of 8 tiles and more on average.
int64_t sink_lists(const JagArgs& a) { return a.sink_list ? a.k_tokens / a.sink_list : a.seqs; }
void sinks_of(JagArgs& a) {
  a.sink_blocks = 0;
  if (!a.seqs || !a.q_tokens || !a.sinks) return;
  const int cell = a.window + 1, rows = a.sinks < cell ? a.sinks : cell;
  const int64_t cells = a.k_tokens / cell;
  const bool fewer_rows = cells * rows < (int64_t)a.seqs * a.sinks, fewer_blocks = cells * ((rows + 31) / 32) < (int64_t)a.seqs * ((a.sinks + 31) / 32);
  a.sink_cell = fewer_rows ? cell : 0, a.sink_rows = fewer_rows ? rows : a.sinks;
  a.sink_list = fewer_blocks ? cell : 0;
  const int64_t lists = sink_lists(a), blocks = ((fewer_blocks ? rows : a.sinks) + 31) / 32, units = lists * blocks * a.hk;
  const int64_t most = a.group * (a.q_tokens / (lists < a.seqs ? lists : a.seqs)) / (8 * 128);
  int64_t shares = 1024 / units;
  shares = shares < most ? shares : most;
  a.sink_shares = (int32_t)(shares > 1 ? shares : 1);
  a.sink_blocks = (int32_t)blocks;
}

// A limit of the interface: first tokens that stay visible are few.
constexpr int kMostSinks = 1024;

struct Space {
  int64_t delta, expo, range, part, sinks, total;
};
Space space_of(JagArgs& a, int dtype, int head_dim, bool gb) {
  sinks_of(a);
  Space s{};
  s.expo = round256(a.q_tokens * a.hq * 4);
  s.range = s.expo + round256(dtype == PDM_F16 ? a.items * 16 * a.hq : 0);
  s.part = s.range + round256(gb ? a.items * 8 : 0);
  s.sinks = s.part + round256(gb ? a.items * a.hq * (part_cols(a) + 2) * 4 : 0);
  s.total = s.sinks + (a.sink_blocks ? (a.sink_cell ? a.k_tokens / a.sink_cell : a.seqs) * a.sink_rows * a.hk * (a.sink_shares + 1) * 2 * head_dim * 4 : 0);
  return s;
}

template <int DT, int D, bool BIAS>
void launch(const JagArgs& a, hipStream_t st) {
  if (a.q_tokens > 0) {
    const int64_t units = a.items * a.hq, most = a.q_tokens > a.seqs ? a.q_tokens : a.seqs;
    const dim3 grid = linear_grid(units + (most + 255) / 256);
    if constexpr (BIAS) {
      if (a.dbias) jag_dq_kernel<DT, D, true, true><<<grid, 256, 0, st>>>(a, units);
      else jag_dq_kernel<DT, D, true, false><<<grid, 256, 0, st>>>(a, units);
    } else {
      jag_dq_kernel<DT, D, false, false><<<grid, 256, 0, st>>>(a, units);
    }
  }
  if (a.dbias) {
    const dim3 grid = linear_grid(a.bias_last / 64 + 1, 1 << 21);  // of columns; heads in between
    jag_dbias_kernel<<<dim3(grid.x, a.hq, grid.y), 1024, 0, st>>>(a);
  }
  if (a.k_tokens > 0) {
    const int64_t items = a.seqs ? a.k_tokens / M + a.seqs : 0, units = items * a.hk, most = a.k_tokens > a.seqs ? a.k_tokens : a.seqs;
    jag_dkv_kernel<DT, D, BIAS, false><<<linear_grid(units + (most + 255) / 256), 256, 0, st>>>(a, units);
    if (a.sink_blocks) {
      const int64_t blocks = sink_lists(a) * a.sink_blocks * a.hk;
      // a workgroup for 256 elements while these are few (512 sequences of 300 tokens with 512 sinks, none of them beyond the window
      // of 1,024, as 610,304 workgroups: the pass took 1,896 us instead of 1,065)
      const int most = (2 * D * (a.sinks < 32 ? a.sinks : 32) + 255) / 256, parts = (int)std::max<int64_t>(1, std::min<int64_t>(most, 8192 / blocks));
      jag_dkv_kernel<DT, D, BIAS, true><<<linear_grid(blocks * a.sink_shares), 256, 0, st>>>(a, blocks * a.sink_shares);
      jag_sinks_kernel<DT, D><<<linear_grid(blocks * parts), 256, 0, st>>>(a, blocks, parts);
    }
  }
}

}  // namespace
}  // namespace pdm

using namespace pdm;

extern "C" int64_t pdm_jagged_attention_bwd_workspace_size(const pdm_jagged_attention_desc* desc, int32_t with_grad_bias) {
  clear_error();
  JagArgs a{};
  if (int e = jag_args(__func__, desc, a)) return e;
  PDM_CHECK_ARG(!with_grad_bias || desc->bias_span > 0, "grad_bias without a bias");
  PDM_CHECK_ARG(a.sinks <= kMostSinks, "at most 1024 sinks in a backward pass");
  return space_of(a, desc->dtype, desc->head_dim, with_grad_bias != 0).total;
}

extern "C" int pdm_jagged_attention_bwd(const pdm_jagged_attention_desc* desc, const void* q, const void* k, const void* v,
                                        const int32_t* cu_q, const int32_t* cu_k, const float* bias, const void* out,
                                        const void* out_rest, const float* stats, const void* grad_out, const float* grad_lse, void* grad_q,
                                        void* grad_k, void* grad_v, float* grad_bias, void* workspace, int64_t workspace_bytes,
                                        pdm_stream_t stream) {
  clear_error();
  JagArgs a{};
  if (int e = jag_args(__func__, desc, a)) return e;
  if (int e = jag_inputs(__func__, a, desc, q, k, v, cu_q, cu_k, bias)) return e;
  PDM_CHECK_ARG(a.sinks <= kMostSinks, "at most 1024 sinks in a backward pass");
  PDM_CHECK_ARG(a.q_tokens == 0 || (out && stats && grad_out && grad_q), "null out / stats / grad_out / grad_q");
  PDM_CHECK_ARG(a.k_tokens == 0 || (grad_k && grad_v), "null grad_k / grad_v");
  PDM_CHECK_ARG(!grad_bias || (bias && (a.q_tokens == 0 || out_rest)), "grad_bias without bias or out_rest");
  for (const void* p : {out, out_rest, grad_out, (const void*)grad_q, (const void*)grad_k, (const void*)grad_v})
    PDM_CHECK_ARG((reinterpret_cast<uintptr_t>(p) & 15) == 0, "outputs and their gradients must be 16-byte aligned");
  const Space sp = space_of(a, desc->dtype, desc->head_dim, grad_bias != nullptr);
  if (sp.total && (!workspace || workspace_bytes < sp.total)) {
    set_error(std::string(__func__) + ": workspace of " + std::to_string(sp.total) + " bytes needed");
    return PDM_ERR_WORKSPACE;
  }
  PDM_CHECK_ARG((reinterpret_cast<uintptr_t>(workspace) & 255) == 0, "workspace must be 256-byte aligned");
  char* ws = static_cast<char*>(workspace);
  a.out = const_cast<void*>(out), a.rest = const_cast<void*>(out_rest), a.stats = const_cast<float*>(stats);
  if (grad_bias && desc->stats_planes == 2) a.outer = a.stats + 2 * a.q_tokens * a.hq;
  a.dout = grad_out, a.dlse = grad_lse, a.dq = grad_q, a.dk = grad_k, a.dv = grad_v, a.dbias = grad_bias;
  a.delta = reinterpret_cast<float*>(ws), a.expo = reinterpret_cast<int32_t*>(ws + sp.expo);
  a.part_range = reinterpret_cast<int32_t*>(ws + sp.range), a.part = reinterpret_cast<float*>(ws + sp.part);
  a.sink_part = reinterpret_cast<float*>(ws + sp.sinks);
  a.part_stride = grad_bias ? part_cols(a) + 2 : 0;
  if (a.q_tokens == 0 && grad_bias) a.items = 0;  // nothing was written that could be summed
  const bool bf16 = desc->dtype == PDM_BF16, biased = bias != nullptr;
  auto run = [&](auto d) {
    constexpr int D = decltype(d)::value;
    if (bf16) biased ? launch<PDM_BF16, D, true>(a, stream) : launch<PDM_BF16, D, false>(a, stream);
    else biased ? launch<PDM_F16, D, true>(a, stream) : launch<PDM_F16, D, false>(a, stream);
  };
  if (desc->head_dim == 64) run(std::integral_constant<int, 64>());
  else run(std::integral_constant<int, 128>());
  PDM_CHECK_LAUNCH();
  return PDM_OK;
}
