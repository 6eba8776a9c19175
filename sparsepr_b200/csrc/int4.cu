// Product of a few rows with 4-bit weights under group scales, and its gradient
// with respect to the rows (layout and formula at spr_int4_linear in the header).
//   y[r][n] = sum_k x[r][k] * (code[n][k] - zero[n][k/group])*scale[n][k/group] + bias[n]
#include "common.cuh"

namespace spr {

namespace {

constexpr int kThreads = 256;
constexpr int kRows = 8;  // rows of x in one pass over the weights

__device__ __forceinline__ float load_as_f32(const void* p, int dtype, int64_t i) {
  if (dtype == SPR_F32) return ((const float*)p)[i];
  if (dtype == SPR_BF16) return to_f32(((const __nv_bfloat16*)p)[i]);
  return to_f32(((const __half*)p)[i]);
}

__device__ __forceinline__ void store_f32(void* p, int dtype, int64_t i, float v) {
  if (dtype == SPR_F32) ((float*)p)[i] = v;
  else if (dtype == SPR_BF16) ((__nv_bfloat16*)p)[i] = __float2bfloat16_rn(v);
  else ((__half*)p)[i] = __float2half_rn(v);
}

// One warp per weight row; a lane takes words of eight codes.
__global__ void __launch_bounds__(kThreads)
int4_linear_kernel(const void* x, int64_t x_stride, int dtype, int64_t rows, int64_t n, int64_t k, int group,
                   const uint32_t* packed, const void* scales, int scale_dtype, const uint8_t* zeros,
                   const void* bias, void* y) {
  const int64_t col = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
  if (col >= n) return;
  const int lane = threadIdx.x & 31;
  const int64_t groups = (k + group - 1) / group, words = groups * group / 8;
  const int64_t r0 = (int64_t)blockIdx.y * kRows;
  const int nr = (int)min((int64_t)kRows, rows - r0);
  float acc[kRows] = {};
  for (int64_t w = lane; w < words; w += 32) {
    const uint32_t word = packed[col * words + w];
    const int64_t g = w * 8 / group;
    const float s = load_as_f32(scales, scale_dtype, col * groups + g);
    const float z = zeros ? (float)zeros[col * groups + g] : 8.f;
    for (int r = 0; r < nr; ++r) {
      float p = 0.f;
      for (int j = 0; j < 8; ++j)
        if (w * 8 + j < k)
          p = fmaf(load_as_f32(x, dtype, (r0 + r) * x_stride + w * 8 + j), ((float)((word >> (4 * j)) & 15) - z) * s, p);
#pragma unroll
      for (int q = 0; q < kRows; ++q)
        if (q == r) acc[q] += p;
    }
  }
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) acc[r] += __shfl_xor_sync(0xffffffffu, acc[r], o);
    if (r < nr && lane == 0)
      store_f32(y, dtype, (r0 + r) * n + col, acc[r] + (bias ? load_as_f32(bias, dtype, col) : 0.f));
  }
}

// One warp per word column (eight k); a lane takes weight rows.
__global__ void __launch_bounds__(kThreads)
int4_linear_grad_kernel(const void* dy, int64_t dy_stride, int dtype, int64_t rows, int64_t n, int64_t k, int group,
                        const uint32_t* packed, const void* scales, int scale_dtype, const uint8_t* zeros, void* dx) {
  const int64_t groups = (k + group - 1) / group, words = groups * group / 8;
  const int64_t w = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
  if (w >= words) return;
  const int lane = threadIdx.x & 31;
  const int64_t g = w * 8 / group, r = blockIdx.y;
  float acc[8] = {};
  for (int64_t col = lane; col < n; col += 32) {
    const uint32_t word = packed[col * words + w];
    const float z = zeros ? (float)zeros[col * groups + g] : 8.f;
    const float d = load_as_f32(dy, dtype, r * dy_stride + col) * load_as_f32(scales, scale_dtype, col * groups + g);
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[j] = fmaf(d, (float)((word >> (4 * j)) & 15) - z, acc[j]);
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) acc[j] += __shfl_xor_sync(0xffffffffu, acc[j], o);
    if (lane == 0 && w * 8 + j < k) store_f32(dx, dtype, r * k + w * 8 + j, acc[j]);
  }
}

int check_int4(const char* what, int64_t stride, int dtype, int64_t rows, int64_t n, int64_t k, int64_t row_len,
               int group, const void* packed, int scale_dtype) {
  if (rows < 0 || n < 0 || k < 1)
    return fail(SPR_ERR_SHAPE, "%s: rows=%lld n=%lld k=%lld", what, (long long)rows, (long long)n, (long long)k);
  if (rows > 65535 || n > 0x7fffffffLL || k > 0x7fffffffLL - (1 << 20))
    return fail(SPR_ERR_SHAPE, "%s: rows=%lld n=%lld k=%lld too large", what, (long long)rows, (long long)n,
                (long long)k);
  if (group < 32 || group % 32 || group > (1 << 20))
    return fail(SPR_ERR_SHAPE, "%s: group=%d must be a multiple of 32", what, group);
  if (rows > 1 && stride < row_len) return fail(SPR_ERR_SHAPE, "%s: row stride %lld", what, (long long)stride);
  for (int d : {dtype, scale_dtype})
    if (d != SPR_F32 && d != SPR_BF16 && d != SPR_F16) return fail(SPR_ERR_DTYPE, "%s: unsupported dtype %d", what, d);
  if (!aligned(packed, 16)) return fail(SPR_ERR_ALIGN, "%s: packed codes must be 16-byte aligned", what);
  return SPR_OK;
}

}  // namespace

}  // namespace spr

using namespace spr;

extern "C" size_t spr_int4_linear_workspace_bytes(int64_t, int64_t, int64_t, int, int) { return 0; }

extern "C" int spr_int4_linear(const void* x, int64_t x_stride, int dtype, int64_t rows, int64_t n, int64_t k,
                               int group, const uint8_t* packed, const void* scales, int scale_dtype,
                               const uint8_t* zeros, const void* bias, void* y, void* workspace,
                               size_t workspace_bytes, void* stream) {
  (void)workspace;
  (void)workspace_bytes;
  if (int rc = check_int4("int4 linear", x_stride, dtype, rows, n, k, k, group, packed, scale_dtype)) return rc;
  if (rows == 0 || n == 0) return SPR_OK;
  if (!x || !packed || !scales || !y) return fail(SPR_ERR_ARG, "int4 linear: null operand");
  const dim3 grid((unsigned)((n + kThreads / 32 - 1) / (kThreads / 32)), (unsigned)((rows + kRows - 1) / kRows));
  int4_linear_kernel<<<grid, kThreads, 0, (cudaStream_t)stream>>>(x, x_stride, dtype, rows, n, k, group,
                                                                  (const uint32_t*)packed, scales, scale_dtype, zeros,
                                                                  bias, y);
  return check_launch("int4 linear");
}

extern "C" size_t spr_int4_linear_grad_workspace_bytes(int64_t, int64_t, int64_t, int, int) { return 0; }

extern "C" int spr_int4_linear_grad(const void* dy, int64_t dy_stride, int dtype, int64_t rows, int64_t n, int64_t k,
                                    int group, const uint8_t* packed, const void* scales, int scale_dtype,
                                    const uint8_t* zeros, void* dx, void* workspace, size_t workspace_bytes,
                                    void* stream) {
  (void)workspace;
  (void)workspace_bytes;
  if (int rc = check_int4("int4 linear grad", dy_stride, dtype, rows, n, k, n, group, packed, scale_dtype)) return rc;
  if (rows == 0) return SPR_OK;
  if (!dx || (n && (!dy || !packed || !scales))) return fail(SPR_ERR_ARG, "int4 linear grad: null operand");
  const int64_t words = (k + group - 1) / group * group / 8;
  const dim3 grid((unsigned)((words + kThreads / 32 - 1) / (kThreads / 32)), (unsigned)rows);
  int4_linear_grad_kernel<<<grid, kThreads, 0, (cudaStream_t)stream>>>(dy, dy_stride, dtype, rows, n, k, group,
                                                                       (const uint32_t*)packed, scales, scale_dtype,
                                                                       zeros, dx);
  return check_launch("int4 linear grad");
}
