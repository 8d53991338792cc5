// Layer norm over the channels of a row (a pixel of an NHWC map, or a token), forward and backward, for fp32, bf16 and fp16
// activations with fp32 parameters:
//   y = (x - mean) * rstd * gamma + beta,  rstd = 1 / sqrt(var + eps)
//   dx = rstd * (h - mean(h) - xh * mean(h * xh)),  h = dy * gamma,  xh = (x - mean) * rstd
//   dgamma += sum over rows of dy * xh,  dbeta += sum over rows of dy
// Statistics and sums are fp32; the variance is the mean of (x - mean)^2, not E[x^2] - mean^2, so that a mean far from zero
// costs no digits.  The only rounding to fewer bits is that of y and dx to the activations' type.
#include "common.h"
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

namespace {

template <typename T> __device__ __forceinline__ float ld(const T* p) { return (float)*p; }
template <> __device__ __forceinline__ float ld<__hip_bfloat16>(const __hip_bfloat16* p) { return __bfloat162float(*p); }
template <> __device__ __forceinline__ float ld<__half>(const __half* p) { return __half2float(*p); }
template <typename T> __device__ __forceinline__ void sto(T* p, float v) { *p = (T)v; }
template <> __device__ __forceinline__ void sto<__hip_bfloat16>(__hip_bfloat16* p, float v) { *p = __float2bfloat16(v); }
template <> __device__ __forceinline__ void sto<__half>(__half* p, float v) { *p = __float2half(v); }

__device__ __forceinline__ float all_sum(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

// one wave per row
template <typename T>
__global__ __launch_bounds__(256) void ln_fwd_kernel(const T* __restrict__ x, int64_t ldx, const float* __restrict__ gamma,
                                                     const float* __restrict__ beta, T* __restrict__ y, float* __restrict__ mean,
                                                     float* __restrict__ rstd, int64_t rows, int C, float eps) {
    const int lane = threadIdx.x & 63;
    for (int64_t r = blockIdx.x * 4ll + (threadIdx.x >> 6); r < rows; r += gridDim.x * 4ll) {
        const T* xr = x + r * ldx;
        float s = 0.f;
        for (int c = lane; c < C; c += 64) s += ld(xr + c);
        const float mu = all_sum(s) / C;
        float q = 0.f;
        for (int c = lane; c < C; c += 64) { const float d = ld(xr + c) - mu; q += d * d; }
        const float is = 1.f / sqrtf(all_sum(q) / C + eps);
        for (int c = lane; c < C; c += 64) {
            const float h = (ld(xr + c) - mu) * is;
            sto(y + r * C + c, fmaf(h, gamma ? gamma[c] : 1.f, beta ? beta[c] : 0.f));
        }
        if (mean && lane == 0) { mean[r] = mu; rstd[r] = is; }
    }
}

template <typename T>
__global__ __launch_bounds__(256) void ln_dx_kernel(const T* __restrict__ dy, int64_t lddy, const T* __restrict__ x, int64_t ldx,
                                                    const float* __restrict__ gamma, const float* __restrict__ mean,
                                                    const float* __restrict__ rstd, T* __restrict__ dx, int64_t rows, int C) {
    const int lane = threadIdx.x & 63;
    for (int64_t r = blockIdx.x * 4ll + (threadIdx.x >> 6); r < rows; r += gridDim.x * 4ll) {
        const T *xr = x + r * ldx, *gr = dy + r * lddy;
        const float mu = mean[r], is = rstd[r];
        float a = 0.f, b = 0.f;
        for (int c = lane; c < C; c += 64) {
            const float h = ld(gr + c) * (gamma ? gamma[c] : 1.f);
            a += h;
            b += h * ((ld(xr + c) - mu) * is);
        }
        a = all_sum(a) / C;
        b = all_sum(b) / C;
        for (int c = lane; c < C; c += 64) {
            const float h = ld(gr + c) * (gamma ? gamma[c] : 1.f);
            sto(dx + r * C + c, is * (h - a - (ld(xr + c) - mu) * is * b));
        }
    }
}

// part[slice][0][c] = sum of dy * xh, part[slice][1][c] = sum of dy over the slice's rows
template <typename T>
__global__ __launch_bounds__(256) void ln_part_kernel(const T* __restrict__ dy, int64_t lddy, const T* __restrict__ x, int64_t ldx,
                                                      const float* __restrict__ mean, const float* __restrict__ rstd,
                                                      float* __restrict__ part, int64_t rows, int C) {
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= C) return;
    float dg = 0.f, db = 0.f;
    for (int64_t r = blockIdx.y; r < rows; r += gridDim.y) {
        const float g = ld(dy + r * lddy + c);
        dg += g * ((ld(x + r * ldx + c) - mean[r]) * rstd[r]);
        db += g;
    }
    part[(blockIdx.y * 2ll) * C + c] = dg;
    part[(blockIdx.y * 2ll + 1) * C + c] = db;
}

// The slices in a fixed order; ONE atomic add per element, so that two launches that share a gradient do not lose either's part.
__global__ __launch_bounds__(256) void ln_fold_kernel(const float* __restrict__ part, int slices, float* __restrict__ dgamma,
                                                      float* __restrict__ dbeta, int C) {
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= C) return;
    float dg = 0.f, db = 0.f;
    for (int s = 0; s < slices; ++s) {
        dg += part[(s * 2ll) * C + c];
        db += part[(s * 2ll + 1) * C + c];
    }
    if (dgamma) atomicAdd(dgamma + c, dg);
    if (dbeta) atomicAdd(dbeta + c, db);
}

int blocks_of(int64_t rows) { const int64_t n = (rows + 3) / 4; return (int)(n < 4096 ? n : 4096); }

template <typename T>
int fwd(const void* x, int64_t ldx, const float* gamma, const float* beta, void* y, float* mean, float* rstd, int64_t rows, int C,
        float eps, hipStream_t st) {
    hipLaunchKernelGGL((ln_fwd_kernel<T>), dim3(blocks_of(rows)), dim3(256), 0, st, (const T*)x, ldx, gamma, beta, (T*)y, mean,
                       rstd, rows, C, eps);
    ADVMIX_CHECK_LAUNCH();
    return ADVMIX_OK;
}

template <typename T>
int bwd(const void* dy, int64_t lddy, const void* x, int64_t ldx, const float* gamma, const float* mean, const float* rstd, void* dx,
        float* dgamma, float* dbeta, float* part, int slices, int64_t rows, int C, hipStream_t st) {
    if (dx)
        hipLaunchKernelGGL((ln_dx_kernel<T>), dim3(blocks_of(rows)), dim3(256), 0, st, (const T*)dy, lddy, (const T*)x, ldx, gamma,
                           mean, rstd, (T*)dx, rows, C);
    if (dgamma || dbeta) {
        hipLaunchKernelGGL((ln_part_kernel<T>), dim3(cdiv(C, 256), slices), dim3(256), 0, st, (const T*)dy, lddy, (const T*)x, ldx,
                           mean, rstd, part, rows, C);
        hipLaunchKernelGGL(ln_fold_kernel, dim3(cdiv(C, 256)), dim3(256), 0, st, part, slices, dgamma, dbeta, C);
    }
    ADVMIX_CHECK_LAUNCH();
    return ADVMIX_OK;
}

bool sizes_ok(int64_t rows, int C, int dtype) {
    return rows >= 1 && C >= 1 && dtype >= ADVMIX_F32 && dtype <= ADVMIX_F16 && rows <= INT64_MAX / 4 / C;
}

}  // namespace

extern "C" int advmix_layer_norm_parts(int64_t rows, int C, int dtype) {
    if (!sizes_ok(rows, C, dtype)) return 0;
    return (int)(rows < 256 ? rows : 256);
}

extern "C" int advmix_layer_norm_fwd(const void* x, int64_t ldx, const float* gamma, const float* beta, void* y, float* mean,
                                     float* rstd, int64_t rows, int C, int dtype, float eps, void* stream) {
    if (!x || !y || ldx < 0 || (mean == nullptr) != (rstd == nullptr) || !(eps >= 0.f) || !sizes_ok(rows, C, dtype))
        return ADVMIX_EINVAL;
    hipStream_t st = (hipStream_t)stream;
    if (dtype == ADVMIX_F32) return fwd<float>(x, ldx, gamma, beta, y, mean, rstd, rows, C, eps, st);
    if (dtype == ADVMIX_BF16) return fwd<__hip_bfloat16>(x, ldx, gamma, beta, y, mean, rstd, rows, C, eps, st);
    return fwd<__half>(x, ldx, gamma, beta, y, mean, rstd, rows, C, eps, st);
}

extern "C" int advmix_layer_norm_bwd(const void* dy, int64_t lddy, const void* x, int64_t ldx, const float* gamma, const float* mean,
                                     const float* rstd, void* dx, float* dgamma, float* dbeta, float* part, int64_t rows, int C,
                                     int dtype, void* stream) {
    if (!dy || !x || !mean || !rstd || ldx < 0 || lddy < 0 || !sizes_ok(rows, C, dtype)) return ADVMIX_EINVAL;
    if ((dgamma || dbeta) && !part) return ADVMIX_EINVAL;
    hipStream_t st = (hipStream_t)stream;
    const int n = advmix_layer_norm_parts(rows, C, dtype);
    if (dtype == ADVMIX_F32) return bwd<float>(dy, lddy, x, ldx, gamma, mean, rstd, dx, dgamma, dbeta, part, n, rows, C, st);
    if (dtype == ADVMIX_BF16)
        return bwd<__hip_bfloat16>(dy, lddy, x, ldx, gamma, mean, rstd, dx, dgamma, dbeta, part, n, rows, C, st);
    return bwd<__half>(dy, lddy, x, ldx, gamma, mean, rstd, dx, dgamma, dbeta, part, n, rows, C, st);
}
