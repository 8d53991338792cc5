// AdamW over the tensors of a model in one flat buffer, moments in 32 or in 8 bits, with the global gradient norm that clips.
//   g' = g * min(1, max_norm / (|g| + 1e-6));  m' = b1 m + (1 - b1) g';  v' = b2 v + (1 - b2) g'^2
//   p' = p - lr wd p - lr / (1 - b1^t) * m' / (sqrt(v' / (1 - b2^t)) + eps)
// The buffer is cut into chunks of up to 1024 elements that belong to one tensor (a table row each: first element, elements,
// group, first block of scales); a workgroup takes a chunk, a wave its 256-element block, a lane four elements.
//
// 8-bit moments: m and r = sqrt(v) as e4m3 codes, per block of 256 one power of two as the scale (exponent byte E: 2^(E - 127)),
// chosen so that the block's largest finite magnitude lies in [128, 256).  A power of two keeps values that do not change on
// the grid when the scale moves.  Rounding: up if the fraction between two codes plus u is 1 or more, u in [0, 1) from a hash of
// the element's place, the step and a seed.  Nearest rounding would freeze r - a step moves it by 0.05 %, half a code is 3 - 6 % -
// while a value that the step hardly moves picks up hardly any noise this way (probability |change| / code distance).  r > 0 is
// held as no less than the smallest code, so that no denominator collapses.
// The moments' arithmetic is rounded operation by operation (no fused multiply-add), so that codes are reproducible from the formula.
#include "common.h"

namespace {

constexpr int HYPER = 8;        // doubles per row: row 0 {max_norm}, row 1 + k {lr, b1, b2, eps, weight decay} of group k
constexpr int COEF = 8;         // floats per row of what a step computes from them

struct Row { int64_t first; int64_t count; int64_t group; int64_t block; };

__device__ __forceinline__ uint32_t mix32(uint32_t x) {
    x ^= x >> 15;
    x *= 0xBB67AE85u;           // 2^32 * frac(sqrt 3), odd
    return x ^ (x >> 13);
}
constexpr uint32_t GOLD = 0x9E3779B9u;      // 2^32 / golden ratio, odd

__global__ __launch_bounds__(256) void sumsq_kernel(const float* __restrict__ g, int64_t n, double* __restrict__ part) {
    double s = 0.0;
    for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < n; i += gridDim.x * 256ll) s += (double)g[i] * (double)g[i];
    __shared__ double red[4];
    s = wave_sum_d(s);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) part[blockIdx.x] = red[0] + red[1] + red[2] + red[3];
}

__device__ double ipow(double b, int64_t t) {                    // b^t by squaring: 2 log2(t) roundings
    double r = 1.0;
    for (; t > 0; t >>= 1, b *= b)
        if (t & 1) r *= b;
    return r;
}

// step += 1 and the step's coefficients per group
__global__ void tick_kernel(const double* __restrict__ hyper, int groups, int64_t* __restrict__ step, const double* __restrict__ part,
                            int nparts, float* __restrict__ norm_out, uint32_t seed, float* __restrict__ coef) {
    const int64_t t = *step + 1;
    __syncthreads();
    float clip = 1.f;
    if (part) {
        double s = 0.0;
        for (int i = 0; i < nparts; ++i) s += part[i];
        const double norm = sqrt(s), c = hyper[0] / (norm + 1e-6);
        clip = c < 1.0 || c != c ? (float)c : 1.f;
        if (threadIdx.x == 0) *norm_out = (float)norm;
    }
    for (int k = threadIdx.x; k < groups; k += blockDim.x) {
        const double* h = hyper + (1 + k) * HYPER;
        float* c = coef + k * COEF;
        c[0] = (float)(h[0] / (1.0 - ipow(h[1], t)));
        c[1] = (float)h[1];
        c[2] = (float)(1.0 - h[1]);
        c[3] = (float)h[2];
        c[4] = (float)(1.0 - h[2]);
        c[5] = (float)(1.0 / sqrt(1.0 - ipow(h[2], t)));
        c[6] = (float)h[3];
        c[7] = (float)(h[0] * h[4]);
    }
    if (threadIdx.x == 0) {
        *step = t;
        coef[groups * COEF] = clip;
        reinterpret_cast<uint32_t*>(coef)[groups * COEF + 1] = mix32((uint32_t)t + mix32(seed * GOLD));
    }
}

struct Coef { float lr1, b1, ob1, b2, ob2, r2, eps, lrwd; };

__device__ __forceinline__ float moment1(float m, float g, const Coef& c) {
#pragma clang fp contract(off)
    return m * c.b1 + g * c.ob1;
}
__device__ __forceinline__ float moment2(float v, float g, const Coef& c) {
#pragma clang fp contract(off)
    return v * c.b2 + (g * g) * c.ob2;
}
__device__ __forceinline__ float scaled(float g, float clip) {
#pragma clang fp contract(off)
    return g * clip;
}
__device__ __forceinline__ float weight(float p, float m, float r, const Coef& c) {
    const float u = m / fmaf(r, c.r2, c.eps);
    return fmaf(-c.lr1, u, fmaf(-c.lrwd, p, p));
}

__global__ __launch_bounds__(256) void adamw_kernel(float* __restrict__ p, const float* __restrict__ g, float* __restrict__ m,
                                                    float* __restrict__ v, const Row* __restrict__ table,
                                                    const float* __restrict__ coef, int groups) {
    const Row row = table[blockIdx.x];
    const int e = threadIdx.x * 4;
    if (e >= row.count) return;
    const int64_t i = row.first + e;
    const Coef c = reinterpret_cast<const Coef*>(coef)[row.group];
    const float clip = coef[groups * COEF];
    f32x4 pv = *reinterpret_cast<f32x4*>(p + i), gv = *reinterpret_cast<const f32x4*>(g + i);
    f32x4 mv = *reinterpret_cast<f32x4*>(m + i), vv = *reinterpret_cast<f32x4*>(v + i);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const float gk = scaled(gv[k], clip);
        mv[k] = moment1(mv[k], gk, c);
        vv[k] = moment2(vv[k], gk, c);
        pv[k] = weight(pv[k], mv[k], sqrtf(vv[k]), c);
    }
    *reinterpret_cast<f32x4*>(p + i) = pv;
    *reinterpret_cast<f32x4*>(m + i) = mv;
    *reinterpret_cast<f32x4*>(v + i) = vv;
}

__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const uint32_t w = __shfl_xor(v, o, 64);
        v = w > v ? w : v;
    }
    return v;
}
__device__ __forceinline__ float pow2(int e) {                   // 2^e for -127 <= e <= 127 (2^-127 is subnormal)
    return e > -127 ? __uint_as_float((uint32_t)(e + 127) << 23) : __uint_as_float(0x00400000u);
}
__device__ __forceinline__ uint32_t finite_bits(float x) {
    const uint32_t b = __float_as_uint(x) & 0x7fffffffu;
    return b < 0x7f800000u ? b : 0u;
}
// exponent byte of a block from the bits of its largest finite magnitude
__device__ __forceinline__ int exponent_byte(uint32_t top) {
    if (top == 0) return 0;
    int e = (int)(top >> 23);                                    // a subnormal top (below 2^-126) clamps to 0 anyway
    e = e - 7;
    return e < 0 ? 0 : e;
}
// e4m3 code of the magnitude z < 256 (already scaled), rounded up where fraction + u16 / 65536 >= 1
__device__ __forceinline__ uint32_t code_of(float z, uint32_t u16) {
    const uint32_t b = __float_as_uint(z);
    const uint32_t big = ((b + (u16 << 4)) >> 20) - ((127 - 7) << 3);
    const float t = z * 512.f, f = floorf(t);                    // below 2^-6: codes are 2^-9 apart
    const uint32_t small = (uint32_t)f + (t - f >= (float)(65536u - u16) * (1.f / 65536.f) ? 1u : 0u);   // (both sides exact)
    return z >= 0.015625f ? big : small;
}
__device__ __forceinline__ float code_value(uint32_t code) {     // magnitude of a code 0 .. 126; 127 is NaN
    const uint32_t e = (code >> 3) & 15u, f = code & 7u;
    const float a = e ? __uint_as_float(((e + 120u) << 23) | (f << 20)) : (float)f * (1.f / 512.f);
    return (code & 127u) == 127u ? __uint_as_float(0x7fc00000u) : a;
}

__device__ __forceinline__ uint32_t pack4(const float (&x)[4], float scale, const uint32_t (&u)[4], uint32_t least) {
    uint32_t w = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const float a = fabsf(x[k]);
        uint32_t c = code_of(a * scale, u[k]);
        if (a > 0.f && c < least) c = least;
        if (!(a < INFINITY)) c = 127u;
        c |= (__float_as_uint(x[k]) >> 31) << 7;
        w |= c << (8 * k);
    }
    return w;
}

__global__ __launch_bounds__(256) void adamw8_kernel(float* __restrict__ p, const float* __restrict__ g, uint8_t* __restrict__ m,
                                                     uint8_t* __restrict__ r, uint8_t* __restrict__ ms, uint8_t* __restrict__ rs,
                                                     const Row* __restrict__ table, const float* __restrict__ coef, int groups) {
    const Row row = table[blockIdx.x];
    const int wave = threadIdx.x >> 6;
    if (wave * 256 >= row.count) return;                         // whole waves
    const int e = threadIdx.x * 4;
    const bool in = e < row.count;
    const int64_t i = row.first + (in ? e : wave * 256);         // lanes past the end read the block's first elements
    const int64_t blk = row.block + wave;
    const Coef c = reinterpret_cast<const Coef*>(coef)[row.group];
    const float clip = coef[groups * COEF];
    const uint32_t key = reinterpret_cast<const uint32_t*>(coef)[groups * COEF + 1];
    const float msc = pow2((int)ms[blk] - 127), rsc = pow2((int)rs[blk] - 127);
    f32x4 pv = *reinterpret_cast<f32x4*>(p + i);
    const f32x4 gv = *reinterpret_cast<const f32x4*>(g + i);
    const uint32_t mw = *reinterpret_cast<const uint32_t*>(m + i), rw = *reinterpret_cast<const uint32_t*>(r + i);
    float mv[4], rv[4];
    uint32_t um[4], ur[4], tm = 0, tr = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const uint32_t mc = mw >> (8 * k), rc = rw >> (8 * k);
        const float a = code_value(mc & 127u) * msc, b = code_value(rc & 127u) * rsc;
        const float gk = scaled(gv[k], clip);
        mv[k] = moment1((mc & 128u) ? -a : a, gk, c);
        rv[k] = sqrtf(moment2(b * b, gk, c));
        pv[k] = weight(pv[k], mv[k], rv[k], c);
        const uint32_t h = mix32((uint32_t)(i + k) * GOLD + key);
        um[k] = h >> 16;
        ur[k] = h & 0xffffu;
        const uint32_t x = in ? finite_bits(mv[k]) : 0u, y = in ? finite_bits(rv[k]) : 0u;
        tm = x > tm ? x : tm;
        tr = y > tr ? y : tr;
    }
    const int em = exponent_byte(wave_max(tm)), er = exponent_byte(wave_max(tr));
    if (in) {
        *reinterpret_cast<f32x4*>(p + i) = pv;
        *reinterpret_cast<uint32_t*>(m + i) = pack4(mv, pow2(127 - em), um, 0u);
        *reinterpret_cast<uint32_t*>(r + i) = pack4(rv, pow2(127 - er), ur, 1u);
    }
    if ((threadIdx.x & 63) == 0) { ms[blk] = (uint8_t)em; rs[blk] = (uint8_t)er; }
}

// fp32 moments <-> codes (root: the codes hold the square root); packing rounds to nearest
__global__ __launch_bounds__(256) void pack8_kernel(const float* __restrict__ x, uint8_t* __restrict__ code, uint8_t* __restrict__ scale,
                                                    const Row* __restrict__ table, int root) {
    const Row row = table[blockIdx.x];
    const int wave = threadIdx.x >> 6;
    if (wave * 256 >= row.count) return;
    const int e = threadIdx.x * 4;
    const bool in = e < row.count;
    float xv[4];
    uint32_t top = 0, half[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const float a = in ? x[row.first + e + k] : 0.f;
        xv[k] = root ? sqrtf(a) : a;
        half[k] = 0x8000u;
        const uint32_t b = finite_bits(xv[k]);
        top = b > top ? b : top;
    }
    const int eb = exponent_byte(wave_max(top));
    if (in) *reinterpret_cast<uint32_t*>(code + row.first + e) = pack4(xv, pow2(127 - eb), half, root ? 1u : 0u);
    if ((threadIdx.x & 63) == 0) scale[row.block + wave] = (uint8_t)eb;
}

__global__ __launch_bounds__(256) void unpack8_kernel(const uint8_t* __restrict__ code, const uint8_t* __restrict__ scale,
                                                      float* __restrict__ x, const Row* __restrict__ table, int root) {
    const Row row = table[blockIdx.x];
    const int e = threadIdx.x * 4;
    if (e >= row.count) return;
    const float s = pow2((int)scale[row.block + (threadIdx.x >> 6)] - 127);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const uint32_t c = code[row.first + e + k];
        float a = code_value(c & 127u) * s;
        a = root ? a * a : ((c & 128u) ? -a : a);
        x[row.first + e + k] = a;
    }
}

bool step_ok(const void* p, const void* g, const void* table, int chunks, const void* hyper, int groups, const void* step,
             const void* part, int nparts, const void* norm_out, const void* coef) {
    return p && g && table && chunks >= 1 && hyper && groups >= 1 && step && coef &&
           (part == nullptr ? nparts == 0 : (nparts >= 1 && norm_out != nullptr));
}

}  // namespace

extern "C" int advmix_grad_sumsq(const float* g, int64_t n, double* part, int nparts, void* stream) {
    if (!g || !part || n < 1 || nparts < 1 || nparts > 65535) return ADVMIX_EINVAL;
    hipLaunchKernelGGL(sumsq_kernel, dim3(nparts), dim3(256), 0, (hipStream_t)stream, g, n, part);
    ADVMIX_CHECK_LAUNCH();
    return ADVMIX_OK;
}

extern "C" int advmix_adamw(float* p, const float* g, float* m, float* v, const int64_t* table, int chunks, const double* hyper,
                            int groups, int64_t* step, const double* part, int nparts, float* norm_out, float* coef, void* stream) {
    if (!step_ok(p, g, table, chunks, hyper, groups, step, part, nparts, norm_out, coef) || !m || !v) return ADVMIX_EINVAL;
    hipStream_t st = (hipStream_t)stream;
    hipLaunchKernelGGL(tick_kernel, dim3(1), dim3(64), 0, st, hyper, groups, step, part, nparts, norm_out, 0u, coef);
    hipLaunchKernelGGL(adamw_kernel, dim3(chunks), dim3(256), 0, st, p, g, m, v, reinterpret_cast<const Row*>(table), coef, groups);
    ADVMIX_CHECK_LAUNCH();
    return ADVMIX_OK;
}

extern "C" int advmix_adamw8(float* p, const float* g, uint8_t* m, uint8_t* r, uint8_t* m_scale, uint8_t* r_scale,
                             const int64_t* table, int chunks, const double* hyper, int groups, int64_t* step, const double* part,
                             int nparts, float* norm_out, int seed, float* coef, void* stream) {
    if (!step_ok(p, g, table, chunks, hyper, groups, step, part, nparts, norm_out, coef) || !m || !r || !m_scale || !r_scale)
        return ADVMIX_EINVAL;
    hipStream_t st = (hipStream_t)stream;
    hipLaunchKernelGGL(tick_kernel, dim3(1), dim3(64), 0, st, hyper, groups, step, part, nparts, norm_out, (uint32_t)seed, coef);
    hipLaunchKernelGGL(adamw8_kernel, dim3(chunks), dim3(256), 0, st, p, g, m, r, m_scale, r_scale,
                       reinterpret_cast<const Row*>(table), coef, groups);
    ADVMIX_CHECK_LAUNCH();
    return ADVMIX_OK;
}

extern "C" int advmix_moments_pack(const float* x, uint8_t* codes, uint8_t* scale, const int64_t* table, int chunks, int root,
                                   void* stream) {
    if (!x || !codes || !scale || !table || chunks < 1) return ADVMIX_EINVAL;
    hipLaunchKernelGGL(pack8_kernel, dim3(chunks), dim3(256), 0, (hipStream_t)stream, x, codes, scale,
                       reinterpret_cast<const Row*>(table), root);
    ADVMIX_CHECK_LAUNCH();
    return ADVMIX_OK;
}

extern "C" int advmix_moments_unpack(const uint8_t* codes, const uint8_t* scale, float* x, const int64_t* table, int chunks, int root,
                                     void* stream) {
    if (!x || !codes || !scale || !table || chunks < 1) return ADVMIX_EINVAL;
    hipLaunchKernelGGL(unpack8_kernel, dim3(chunks), dim3(256), 0, (hipStream_t)stream, codes, scale, x,
                       reinterpret_cast<const Row*>(table), root);
    ADVMIX_CHECK_LAUNCH();
    return ADVMIX_OK;
}
