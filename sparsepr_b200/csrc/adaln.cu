// Modulated layer norm with an optional gated residual in front of it, forward
// and backward (the operands are described at SprAdaln in the header):
//   z = x + gate*y,  n = (z - mean z) * rstd,  h = n*w + shift,  w = offset + scale
//   u = dh*w,  g = dz + rstd*(u - mean u - n*mean(u*n)),  dx = g,  dy = g*gate
//   dshift = sum dh,  dscale = sum dh*n,  dgate = sum g*y   over the rows of a group
// Statistics and sums are fp32; the variance is taken about the mean, in a
// second pass over the row.
#include "common.cuh"

namespace spr {

namespace {

constexpr int kRowThreads = 256;
constexpr int kMaxChannels = 16384;

template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }

template <int N>
__device__ __forceinline__ void block_sum(float (&v)[N], float (*red)[32]) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
  __syncthreads();  // the buffer's last readers are done
  if (lane == 0)
#pragma unroll
    for (int i = 0; i < N; ++i) red[i][warp] = v[i];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    v[i] = 0.f;
    for (int w = 0; w < (int)blockDim.x / 32; ++w) v[i] += red[i][w];
  }
}

// The residual stream: product and sum rounded to fp32 one after the other, so
// that z is what the two separate operations store.
template <typename T>
__device__ __forceinline__ float residual(float x, float y, float gate) {
  return to_f32(from_f32<T>(__fadd_rn(x, __fmul_rn(gate, y))));
}

template <typename T, typename MT>
__global__ void __launch_bounds__(kRowThreads) adaln_forward_kernel(const SprAdaln op) {
  __shared__ float red[1][32];
  const int64_t row = blockIdx.x, b = row / op.tokens, t = row % op.tokens;
  const int c = op.channels;
  const T* x = (const T*)op.x + b * op.x_sb + t * op.x_st;
  const T* y = (const T*)op.y + (op.y ? b * op.y_sb + t * op.y_st : 0);
  const MT* gate = (const MT*)op.gate + (op.gate ? b * op.gate_sb + t * op.gate_st : 0);
  const MT* scale = (const MT*)op.scale + (op.scale ? b * op.scale_sb + t * op.scale_st : 0);
  const MT* shift = (const MT*)op.shift + (op.shift ? b * op.shift_sb + t * op.shift_st : 0);
  auto at = [&](int i) {
    return op.y ? residual<T>(to_f32(x[i]), to_f32(y[i]), op.gate ? to_f32(gate[i]) : 1.f) : to_f32(x[i]);
  };
  float s[1] = {0.f};
  for (int i = threadIdx.x; i < c; i += kRowThreads) s[0] += at(i);
  block_sum(s, red);
  const float mean = s[0] / c;
  s[0] = 0.f;
  for (int i = threadIdx.x; i < c; i += kRowThreads) {
    const float d = at(i) - mean;
    s[0] = fmaf(d, d, s[0]);
  }
  block_sum(s, red);
  const float rstd = rsqrtf(s[0] / c + op.eps);
  for (int i = threadIdx.x; i < c; i += kRowThreads) {
    const float z = at(i);
    if (op.y) ((T*)op.z)[row * c + i] = from_f32<T>(z);
    const float w = op.scale ? op.scale_offset + to_f32(scale[i]) : 1.f;
    ((T*)op.h)[row * c + i] = from_f32<T>(fmaf((z - mean) * rstd, w, op.shift ? to_f32(shift[i]) : 0.f));
  }
  if (threadIdx.x == 0 && op.mean) {
    op.mean[row] = mean;
    op.rstd[row] = rstd;
  }
}

// dx and dy of one row per CTA, and the row's two means for the column sums.
template <typename T, typename MT>
__global__ void __launch_bounds__(kRowThreads)
adaln_backward_rows_kernel(const SprAdaln op, const SprAdalnGrad gr, float* means) {
  __shared__ float red[2][32];
  const int64_t row = blockIdx.x, b = row / op.tokens, t = row % op.tokens;
  const int c = op.channels;
  const T* z = (const T*)op.x + b * op.x_sb + t * op.x_st;
  const T* dh = (const T*)gr.dh + b * gr.dh_sb + t * gr.dh_st;
  const T* dz = (const T*)gr.dz + (gr.dz ? b * gr.dz_sb + t * gr.dz_st : 0);
  const MT* gate = (const MT*)op.gate + (op.gate ? b * op.gate_sb + t * op.gate_st : 0);
  const MT* scale = (const MT*)op.scale + (op.scale ? b * op.scale_sb + t * op.scale_st : 0);
  const float mean = op.mean[row], rstd = op.rstd[row];
  float s[2] = {0.f, 0.f};
  for (int i = threadIdx.x; i < c; i += kRowThreads) {
    const float u = to_f32(dh[i]) * (op.scale ? op.scale_offset + to_f32(scale[i]) : 1.f);
    s[0] += u;
    s[1] = fmaf(u, (to_f32(z[i]) - mean) * rstd, s[1]);
  }
  block_sum(s, red);
  const float m0 = s[0] / c, m1 = s[1] / c;
  for (int i = threadIdx.x; i < c; i += kRowThreads) {
    const float u = to_f32(dh[i]) * (op.scale ? op.scale_offset + to_f32(scale[i]) : 1.f);
    const float n = (to_f32(z[i]) - mean) * rstd;
    const float g = fmaf(rstd, u - m0 - n * m1, gr.dz ? to_f32(dz[i]) : 0.f);
    ((T*)gr.dx)[row * c + i] = from_f32<T>(g);
    if (gr.dy) ((T*)gr.dy)[row * c + i] = from_f32<T>(g * (op.gate ? to_f32(gate[i]) : 1.f));
  }
  if (threadIdx.x == 0) {
    means[2 * row] = m0;
    means[2 * row + 1] = m1;
  }
}

// Column sums over the rows of a group, one thread per column.
template <typename T, typename MT>
__global__ void __launch_bounds__(kRowThreads)
adaln_backward_columns_kernel(const SprAdaln op, const SprAdalnGrad gr, const float* means) {
  const int i = blockIdx.y * kRowThreads + threadIdx.x;
  const int c = op.channels;
  if (i >= c) return;
  const int64_t group = blockIdx.x;
  const int64_t b0 = gr.mod_batch ? (gr.mod_tokens ? group / op.tokens : group) : 0;
  const int64_t t0 = gr.mod_tokens ? group % op.tokens : 0;
  const int64_t nb = gr.mod_batch ? 1 : op.batch, nt = gr.mod_tokens ? 1 : op.tokens;
  float dshift = 0.f, dscale = 0.f, dgate = 0.f;
  for (int64_t b = b0; b < b0 + nb; ++b)
    for (int64_t t = t0; t < t0 + nt; ++t) {
      const int64_t row = b * op.tokens + t;
      const float mean = op.mean[row], rstd = op.rstd[row];
      const float dh = to_f32(((const T*)gr.dh)[b * gr.dh_sb + t * gr.dh_st + i]);
      const float n = (to_f32(((const T*)op.x)[b * op.x_sb + t * op.x_st + i]) - mean) * rstd;
      dshift += dh;
      dscale = fmaf(dh, n, dscale);
      if (gr.dgate) {
        const float w =
            op.scale ? op.scale_offset + to_f32(((const MT*)op.scale)[b * op.scale_sb + t * op.scale_st + i]) : 1.f;
        const float dz = gr.dz ? to_f32(((const T*)gr.dz)[b * gr.dz_sb + t * gr.dz_st + i]) : 0.f;
        const float g = fmaf(rstd, dh * w - means[2 * row] - n * means[2 * row + 1], dz);
        dgate = fmaf(g, to_f32(((const T*)op.y)[b * op.y_sb + t * op.y_st + i]), dgate);
      }
    }
  if (gr.dshift) ((MT*)gr.dshift)[group * c + i] = from_f32<MT>(dshift);
  if (gr.dscale) ((MT*)gr.dscale)[group * c + i] = from_f32<MT>(dscale);
  if (gr.dgate) ((MT*)gr.dgate)[group * c + i] = from_f32<MT>(dgate);
}

int check_adaln(const SprAdaln* op) {
  if (!op) return fail(SPR_ERR_ARG, "adaln: no operands");
  if (op->batch < 0 || op->tokens < 0 || op->channels < 1 || op->channels > kMaxChannels)
    return fail(SPR_ERR_SHAPE, "adaln: batch=%lld tokens=%lld channels=%d (channels must be 1..%d)",
                (long long)op->batch, (long long)op->tokens, op->channels, kMaxChannels);
  if (op->tokens && op->batch > 0x7fffffffLL / op->tokens) return fail(SPR_ERR_SHAPE, "adaln: batch*tokens too large");
  if (op->dtype != SPR_F32 && op->dtype != SPR_BF16 && op->dtype != SPR_F16)
    return fail(SPR_ERR_DTYPE, "adaln: unsupported dtype %d", op->dtype);
  if (op->mod_dtype != op->dtype && op->mod_dtype != SPR_F32)
    return fail(SPR_ERR_DTYPE, "adaln: shift/scale/gate dtype %d must be the element type %d or fp32", op->mod_dtype,
                op->dtype);
  if (op->gate && !op->y) return fail(SPR_ERR_ARG, "adaln: a gate without a branch");
  return SPR_OK;
}

// Calls f(T{}, MT{}) for the operands' types.
template <typename F>
int by_type(const SprAdaln* op, F f) {
  if (op->dtype == SPR_F32) return f(float{}, float{});
  if (op->dtype == SPR_BF16)
    return op->mod_dtype == SPR_F32 ? f(__nv_bfloat16{}, float{}) : f(__nv_bfloat16{}, __nv_bfloat16{});
  return op->mod_dtype == SPR_F32 ? f(__half{}, float{}) : f(__half{}, __half{});
}

}  // namespace

}  // namespace spr

using namespace spr;

extern "C" int spr_adaln_forward(const SprAdaln* op, void* stream) {
  if (int rc = check_adaln(op)) return rc;
  const int64_t rows = op->batch * op->tokens;
  if (rows == 0) return SPR_OK;
  if (!op->x || !op->h || (op->y && !op->z)) return fail(SPR_ERR_ARG, "adaln forward: null operand");
  return by_type(op, [&](auto t, auto m) {
    using T = decltype(t);
    using MT = decltype(m);
    adaln_forward_kernel<T, MT><<<(unsigned)rows, kRowThreads, 0, (cudaStream_t)stream>>>(*op);
    return check_launch("adaln forward");
  });
}

extern "C" size_t spr_adaln_backward_workspace_bytes(int64_t batch, int64_t tokens, int channels, int mod_batch,
                                                     int mod_tokens) {
  (void)channels;
  (void)mod_batch;
  (void)mod_tokens;
  return (size_t)std::max<int64_t>(batch * tokens, 0) * 2 * sizeof(float);
}

extern "C" int spr_adaln_backward(const SprAdaln* op, const SprAdalnGrad* grad, void* workspace, size_t workspace_bytes,
                                  void* stream) {
  if (int rc = check_adaln(op)) return rc;
  if (!grad) return fail(SPR_ERR_ARG, "adaln backward: no gradients");
  const int64_t rows = op->batch * op->tokens;
  if (rows == 0) return SPR_OK;
  if (!op->x || !op->mean || !op->rstd || !grad->dh || !grad->dx || (grad->dgate && !op->y))
    return fail(SPR_ERR_ARG, "adaln backward: null operand");
  const size_t need =
      spr_adaln_backward_workspace_bytes(op->batch, op->tokens, op->channels, grad->mod_batch, grad->mod_tokens);
  if (!workspace || workspace_bytes < need)
    return fail(SPR_ERR_WORKSPACE, "adaln backward: workspace %zu < %zu bytes", workspace_bytes, need);
  const int64_t groups = (grad->mod_batch ? op->batch : 1) * (grad->mod_tokens ? op->tokens : 1);
  return by_type(op, [&](auto t, auto m) {
    using T = decltype(t);
    using MT = decltype(m);
    cudaStream_t st = (cudaStream_t)stream;
    adaln_backward_rows_kernel<T, MT><<<(unsigned)rows, kRowThreads, 0, st>>>(*op, *grad, (float*)workspace);
    if (grad->dshift || grad->dscale || grad->dgate)
      adaln_backward_columns_kernel<T, MT>
          <<<dim3((unsigned)groups, (op->channels + kRowThreads - 1) / kRowThreads), kRowThreads, 0, st>>>(
              *op, *grad, (const float*)workspace);
    return check_launch("adaln backward");
  });
}
