// A table of buckets spread over distances, and its gradient.
//
// Bound by the bytes of the [heads, span] side and, when small, by launches.  Forward: a thread per column and 4 heads.  Backward:
// a workgroup per (bucket, head) sums the columns that are its own, in a fixed order and in 64 bits; in large maps one workgroup
// finds the first and last column of every bucket before (a bucket's columns are neighbours in all but odd maps).  Eight reads of
// the map are on their way before the first is looked at: 65,536 columns of 64 heads in one bucket take 40 us instead of 71 (both
// launches, back to back), in 320 logarithmic ones 32 either way (13.8 for the ranges, 23.4 for the sums, by themselves).
#include "pdm_common.h"

namespace pdm {
namespace {

constexpr int kBuckets = 8192;

// Up to so many reads of the map every (bucket, head) looks at all of it, in one launch less; above, at its bucket's columns.  32
// buckets, 64 heads, us without and with ranges: 4,097 columns 5.4 and 6.4, 32,768 21.9 and 19.1; 512 buckets, 16 heads: 300
// columns 7.3 and 9.5, 8,193 20.4 and 11.4.
constexpr int64_t kWhole = 24 << 20;

template <int DT>
__device__ __forceinline__ float table_value(const void* t, int64_t i) {
  if constexpr (DT == PDM_F32) return static_cast<const float*>(t)[i];
  else if constexpr (DT == PDM_BF16) return bf16_bits_to_f32(static_cast<const uint16_t*>(t)[i]);
  else return f16_bits_to_f32(static_cast<const uint16_t*>(t)[i]);
}

template <int DT>
__global__ void __launch_bounds__(256) bucket_bias_kernel(const void* table, int buckets, int heads, const int32_t* map, int span, float* out) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= span) return;
  const int b = map[c];
  const bool ok = (uint32_t)b < (uint32_t)buckets;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int h = blockIdx.y * 4 + i;
    if (h < heads) out[(int64_t)h * span + c] = ok ? table_value<DT>(table, (int64_t)b * heads + h) : 0.0f;
  }
}

// range[2 b], range[2 b + 1]: first and last column of bucket b (first > last: none)
__global__ void __launch_bounds__(1024) bucket_range_kernel(const int32_t* map, int span, int buckets, int32_t* range) {
  __shared__ int lo[kBuckets], hi[kBuckets];
  for (int b = threadIdx.x; b < buckets; b += 1024) lo[b] = 0x7fffffff, hi[b] = -1;
  __syncthreads();
  // a bucket's first and last column are ends of runs of one bucket, and these are few
  const int lane = threadIdx.x & 63;
  for (int c0 = threadIdx.x; c0 < (span + 63 & ~63); c0 += 8 * 1024) {  // (whole waves)
    int m[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int c = c0 + 1024 * i;
      m[i] = c < span ? map[c] : -1;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int c = c0 + 1024 * i, b = m[i], before = __shfl_up(b, 1), behind = __shfl_down(b, 1);
      if ((uint32_t)b < (uint32_t)buckets) {
        if (lane == 0 || b != before) atomicMin(&lo[b], c);
        if (lane == 63 || b != behind) atomicMax(&hi[b], c);
      }
    }
  }
  __syncthreads();
  for (int b = threadIdx.x; b < buckets; b += 1024) range[2 * b] = lo[b], range[2 * b + 1] = hi[b];
}

__global__ void __launch_bounds__(256) bucket_grad_kernel(const float* grad, const int32_t* map, int span, int heads, const int32_t* range,
                                                          int dtype, void* out) {
  __shared__ double part[4];
  const int b = blockIdx.x, h = blockIdx.y, lo = range ? range[2 * b] : 0, hi = range ? range[2 * b + 1] : span - 1;
  double sum = 0.0;
  for (int c0 = lo; c0 <= hi; c0 += 8 * 256) {
    int m[8];
    float g[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) m[i] = c0 + 256 * i + (int)threadIdx.x <= hi ? map[c0 + 256 * i + threadIdx.x] : -1;
#pragma unroll
    for (int i = 0; i < 8; ++i) g[i] = m[i] == b ? grad[(int64_t)h * span + c0 + 256 * i + threadIdx.x] : 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += g[i];
  }
  for (int o = 1; o < 64; o <<= 1) sum += __shfl_xor(sum, o);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x) return;
  const float v = (float)((part[0] + part[1]) + (part[2] + part[3]));
  const int64_t at = (int64_t)b * heads + h;
  if (dtype == PDM_F32) static_cast<float*>(out)[at] = v;
  else static_cast<uint16_t*>(out)[at] = (uint16_t)(dtype == PDM_BF16 ? f32_to_bf16_bits(v) : f32_to_f16_bits(v));
}

int check(const char* fn, int32_t dtype, int32_t buckets, int32_t heads, int32_t span) {
  auto bad = [&](const char* m) {
    set_error(std::string(fn) + ": " + m);
    return (int)PDM_ERR_INVALID;
  };
  if (dtype != PDM_F32 && dtype != PDM_F16 && dtype != PDM_BF16) return bad("dtype must be F32, F16 or BF16");
  if (buckets < 1 || buckets > kBuckets) return bad("num_buckets must lie in [1, 8192]");
  if (heads < 1 || heads > 65535) return bad("heads must lie in [1, 65535]");
  if (span < 1 || span > (1 << 24)) return bad("span must lie in [1, 2^24]");
  return PDM_OK;
}

}  // namespace
}  // namespace pdm

using namespace pdm;

extern "C" int pdm_bucket_bias_fwd(const void* table, int32_t dtype, int32_t num_buckets, int32_t heads, const int32_t* buckets,
                                   int32_t span, float* out, pdm_stream_t stream) {
  clear_error();
  if (int e = check(__func__, dtype, num_buckets, heads, span)) return e;
  PDM_CHECK_ARG(table && buckets && out, "null table / buckets / out");
  const dim3 grid((span + 255) / 256, (heads + 3) / 4);
  if (dtype == PDM_F32) bucket_bias_kernel<PDM_F32><<<grid, 256, 0, stream>>>(table, num_buckets, heads, buckets, span, out);
  else if (dtype == PDM_BF16) bucket_bias_kernel<PDM_BF16><<<grid, 256, 0, stream>>>(table, num_buckets, heads, buckets, span, out);
  else bucket_bias_kernel<PDM_F16><<<grid, 256, 0, stream>>>(table, num_buckets, heads, buckets, span, out);
  PDM_CHECK_LAUNCH();
  return PDM_OK;
}

extern "C" int pdm_bucket_bias_bwd(const float* grad_out, const int32_t* buckets, int32_t span, int32_t num_buckets, int32_t heads,
                                   int32_t dtype, void* grad_table, void* workspace, int64_t workspace_bytes, pdm_stream_t stream) {
  clear_error();
  if (int e = check(__func__, dtype, num_buckets, heads, span)) return e;
  PDM_CHECK_ARG(grad_out && buckets && grad_table, "null grad_out / buckets / grad_table");
  PDM_CHECK_ARG((reinterpret_cast<uintptr_t>(workspace) & 3) == 0, "workspace must be 4-byte aligned");
  if (!workspace || workspace_bytes < 8 * (int64_t)num_buckets) {
    set_error(std::string(__func__) + ": workspace of " + std::to_string(8 * (int64_t)num_buckets) + " bytes needed");
    return PDM_ERR_WORKSPACE;
  }
  int32_t* range = (int64_t)num_buckets * heads * span > kWhole ? static_cast<int32_t*>(workspace) : nullptr;
  if (range) bucket_range_kernel<<<1, 1024, 0, stream>>>(buckets, span, num_buckets, range);
  bucket_grad_kernel<<<dim3(num_buckets, heads), 256, 0, stream>>>(grad_out, buckets, span, heads, range, dtype, grad_table);
  PDM_CHECK_LAUNCH();
  return PDM_OK;
}
