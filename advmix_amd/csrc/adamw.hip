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
// while a value that the step hardly moves picks up hardly any noise this way (probability |change| / code distance).  600 steps
// of the formulas over 4096 elements, b2 = 0.999: the average of r^2 stays within 4 % of v's (one element's spreads by up to 36 %)
// and the weights' path within 14 %; with nearest rounding r^2 is 36 - 54 % low and the path 33 % off.  r > 0 is held as no less
// than the smallest code, so that no denominator collapses.
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

// Squares in fp64: fp32 ones overflow at 1.8e19 and vanish below 1e-23.  63.6 M elements 46 us = 5.5 TB/s (one 4-byte load in
// flight a lane: 111 us).
__global__ __launch_bounds__(256) void sumsq_kernel(const float* __restrict__ g, int64_t n, double* __restrict__ part) {
    const int64_t quads = n >> 2, step = gridDim.x * 256ll;
    double s[4] = {0.0, 0.0, 0.0, 0.0};
    int64_t i = blockIdx.x * 256ll + threadIdx.x;
    const f32x4* q = reinterpret_cast<const f32x4*>(g);
    for (; i + 3 * step < quads; i += 4 * step) {                // four loads in flight
        f32x4 w[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) w[u] = q[i + u * step];
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[e] = fma((double)w[u][e], (double)w[u][e], s[e]);
    }
    for (; i < quads; i += step) {
        const f32x4 w = q[i];
#pragma unroll
        for (int e = 0; e < 4; ++e) s[e] = fma((double)w[e], (double)w[e], s[e]);
    }
    if (blockIdx.x == 0 && threadIdx.x < (n & 3)) {
        const double w = g[4 * quads + threadIdx.x];
        s[0] = fma(w, w, s[0]);
    }
    __shared__ double red[4];
    const double t = wave_sum_d((s[0] + s[1]) + (s[2] + s[3]));
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = t;
    __syncthreads();
    if (threadIdx.x == 0) part[blockIdx.x] = (red[0] + red[1]) + (red[2] + red[3]);
}

__device__ double ipow(double b, int64_t t) {                    // b^t by squaring: 2 log2(t) roundings
    double r = 1.0;
    for (; t > 0; t >>= 1, b *= b)
        if (t & 1) r *= b;
    return r;
}

struct Coef { float lr1, b1, ob1, b2, ob2, r2, eps, lrwd; };
// What a step needs of the optimizer's settings; ``coef`` (device scratch) holds a Coef per group, then clip, key and a ticket.
struct Step {
    const double* hyper;
    int groups;
    int64_t* step;
    const double* part;
    int nparts;
    float* norm_out;
    uint32_t seed;
    float* coef;
};

__device__ __forceinline__ float step_size(const double* h, int64_t t) { return (float)(h[0] / (1.0 - ipow(h[1], t))); }
__device__ __forceinline__ float root_scale(const double* h, int64_t t) { return (float)(1.0 / sqrt(1.0 - ipow(h[2], t))); }
__device__ __forceinline__ void plain_coefs(Coef& c, const double* h) {
    c.b1 = (float)h[1];
    c.ob1 = (float)(1.0 - h[1]);
    c.b2 = (float)h[2];
    c.ob2 = (float)(1.0 - h[2]);
    c.eps = (float)h[3];
    c.lrwd = (float)(h[0] * h[4]);
}
// The norm's parts, by 256 threads, in red[4]; a barrier has to follow.
__device__ __forceinline__ void add_parts(const Step& s, double* red) {
    double v = 0.0;
    for (int i = threadIdx.x; i < s.nparts; i += 256) v += s.part[i];
    v = wave_sum_d(v);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
}
__device__ __forceinline__ float clip_of(const Step& s, const double* red, bool tell) {
    const double norm = sqrt((red[0] + red[1]) + (red[2] + red[3])), c = s.hyper[0] / (norm + 1e-6);
    if (tell) *s.norm_out = (float)norm;
    return c < 1.0 || c != c ? (float)c : 1.f;
}
__device__ __forceinline__ uint32_t key_of(const Step& s, int64_t t) { return mix32((uint32_t)t + mix32(s.seed * GOLD)); }

// step += 1 and the step's coefficients per group (one workgroup)
__global__ __launch_bounds__(256) void tick_kernel(Step s) {
    __shared__ double red[4];
    const int64_t t = *s.step + 1;
    if (s.part) add_parts(s, red);
    __syncthreads();                                             // (also: everyone has read *step)
    for (int k = threadIdx.x; k < s.groups; k += 256) {
        const double* h = s.hyper + (1 + k) * HYPER;
        Coef c;
        plain_coefs(c, h);
        c.lr1 = step_size(h, t);
        c.r2 = root_scale(h, t);
        reinterpret_cast<Coef*>(s.coef)[k] = c;
    }
    if (threadIdx.x == 0) {
        float* c = s.coef + s.groups * COEF;
        c[0] = s.part ? clip_of(s, red, true) : 1.f;
        reinterpret_cast<uint32_t*>(c)[1] = key_of(s, t);
        *s.step = t;
    }
}

// The coefficients a workgroup of the step needs: OWN: worked out by itself, without the launch before; the last workgroup to have
// read the step counter moves it on (and puts the ticket back).  Every thread of the workgroup comes here.
template <bool OWN> __device__ __forceinline__ void settings(const Step& s, int64_t group, Coef& c, float& clip, uint32_t& key) {
    if (!OWN) {
        c = reinterpret_cast<const Coef*>(s.coef)[group];
        clip = s.coef[s.groups * COEF];
        key = reinterpret_cast<const uint32_t*>(s.coef)[s.groups * COEF + 1];
        return;
    }
    __shared__ double red[4];
    __shared__ Coef mine;
    __shared__ float by;
    __shared__ uint32_t k;
    const double* h = s.hyper + (1 + group) * HYPER;
    if (s.part) add_parts(s, red);
    const int64_t t = *s.step + 1;
    if (threadIdx.x == 0) mine.lr1 = step_size(h, t);
    if (threadIdx.x == 64) mine.r2 = root_scale(h, t);
    if (threadIdx.x == 128) {
        Coef q;
        plain_coefs(q, h);
        mine.b1 = q.b1; mine.ob1 = q.ob1; mine.b2 = q.b2; mine.ob2 = q.ob2; mine.eps = q.eps; mine.lrwd = q.lrwd;
    }
    if (threadIdx.x == 192) k = key_of(s, t);
    __syncthreads();                                             // everyone here has read *step
    if (threadIdx.x == 0) {
        by = s.part ? clip_of(s, red, blockIdx.x == 0) : 1.f;
        uint32_t* ticket = reinterpret_cast<uint32_t*>(s.coef) + s.groups * COEF + 2;
        if (atomicAdd(ticket, 1u) == gridDim.x - 1) {
            *ticket = 0u;
            *s.step = t;
        }
    }
    __syncthreads();
    c = mine;
    clip = by;
    key = k;
}

// sqrt, off by at most one place, or rounded to nearest (EXACT: the remainders of the neighbours say which it is).  The instruction
// takes no subnormal numbers and the remainders of tiny ones vanish: below 2^-96 it works on v * 2^64.
template <bool EXACT> __device__ __forceinline__ float root(float v) {
    const int up = v < 0x1p-96f ? 32 : 0;
    const float w = __builtin_amdgcn_ldexpf(v, 2 * up);
    float s = __builtin_amdgcn_sqrtf(w);
    if (EXACT) {
        const float lo = __uint_as_float(__float_as_uint(s) - 1u), hi = __uint_as_float(__float_as_uint(s) + 1u);
        const float a = fmaf(-lo, s, w), b = fmaf(-hi, s, w);
        s = a <= 0.f ? lo : s;
        s = b > 0.f ? hi : s;                                    // (0, infinity and NaN: both comparisons are false)
    }
    return __builtin_amdgcn_ldexpf(s, -up);
}

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
    const float u = m * __builtin_amdgcn_rcpf(fmaf(r, c.r2, c.eps));     // (1 ulp; eps keeps it away from subnormals)
    return fmaf(-c.lr1, u, fmaf(-c.lrwd, p, p));
}

// NT: the step's data is larger than the last-level cache (256 MB), so it goes past the caches in both directions; see stream_past.
template <bool NT, typename T> __device__ __forceinline__ T ldv(const T* p) {
    return NT ? __builtin_nontemporal_load(p) : *p;
}
template <bool NT, typename T> __device__ __forceinline__ void stv(T* p, T v) {
    if (NT) __builtin_nontemporal_store(v, p);
    else *p = v;
}
__device__ __forceinline__ const f32x4* quad(const float* p) { return reinterpret_cast<const f32x4*>(p); }
__device__ __forceinline__ f32x4* quad(float* p) { return reinterpret_cast<f32x4*>(p); }

// Bound by memory: 28 bytes an element, 28.5 M elements in 300 tensors 138 us = 5.8 TB/s (in 30 tensors 131 us).  A workgroup takes one
// chunk and ends (walking workgroups with the next chunk on its way are slower: through the caches 170 us with 2048 of them, 151 us
// this way).
template <bool NT, bool OWN>
__global__ __launch_bounds__(256) void adamw_kernel(float* __restrict__ p, const float* __restrict__ g, float* __restrict__ m,
                                                    float* __restrict__ v, const Row* __restrict__ table, Step step) {
    const Row row = table[blockIdx.x];
    const int e = threadIdx.x * 4;
    const bool in = e < row.count;
    if (!OWN && !in) return;
    const int64_t i = row.first + (in ? e : 0);
    f32x4 pv = ldv<NT>(quad(p + i));
    const f32x4 gv = ldv<NT>(quad(g + i));
    f32x4 mv = ldv<NT>(quad(m + i)), vv = ldv<NT>(quad(v + i));
    Coef k;
    float clip;
    uint32_t key;
    settings<OWN>(step, row.group, k, clip, key);
    if (!in) return;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float gj = scaled(gv[j], clip);
        mv[j] = moment1(mv[j], gj, k);
        vv[j] = moment2(vv[j], gj, k);
        pv[j] = weight(pv[j], mv[j], root<false>(vv[j]), k);
    }
    stv<NT>(quad(p + i), pv);
    stv<NT>(quad(m + i), mv);
    stv<NT>(quad(v + i), vv);
}

// Maximum over the wave, in every lane (the permutations of a butterfly: lane ^ 1, lane ^ 2, mirrors of 8 and 16, rows, halves)
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
template <int CTRL> __device__ __forceinline__ uint32_t dpp(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, CTRL, 0xf, 0xf, true);
}
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
    v = max(v, dpp<0xB1>(v));
    v = max(v, dpp<0x4E>(v));
    v = max(v, dpp<0x141>(v));
    v = max(v, dpp<0x140>(v));
    u32x2 s = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = max(s[0], s[1]);
    s = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return (uint32_t)__builtin_amdgcn_readfirstlane((int)max(s[0], s[1]));
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
typedef float f32x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ void decode(float (&x)[4], uint32_t w) {      // four e4m3 codes
    const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    x[0] = a[0]; x[1] = a[1]; x[2] = b[0]; x[3] = b[1];
}
// Four codes of x * scale (below 256 in magnitude): the conversion adds the upper 20 bits of ``u`` to the fraction between two
// codes and drops the rest, which is the rule above for u = 16 bits / 2^16, exact below the normal range too.
__device__ __forceinline__ uint32_t encode(const float (&x)[4], float scale, const uint32_t (&u)[4]) {
    int w = __builtin_amdgcn_cvt_sr_fp8_f32(x[0] * scale, u[0], 0, 0);
    w = __builtin_amdgcn_cvt_sr_fp8_f32(x[1] * scale, u[1], w, 1);
    w = __builtin_amdgcn_cvt_sr_fp8_f32(x[2] * scale, u[2], w, 2);
    return (uint32_t)__builtin_amdgcn_cvt_sr_fp8_f32(x[3] * scale, u[3], w, 3);
}
// r > 0 is held as no less than the smallest code; only where the scaled value is below it can the code be 0
__device__ __forceinline__ uint32_t at_least_one(uint32_t w, const float (&r)[4]) {
#pragma unroll
    for (int k = 0; k < 4; ++k)
        if (r[k] > 0.f && !(w & (255u << 8 * k))) w |= 1u << 8 * k;
    return w;
}
// NaN for what is not finite
__device__ __forceinline__ uint32_t poison(uint32_t w, const float (&x)[4]) {
#pragma unroll
    for (int k = 0; k < 4; ++k)
        if (!(fabsf(x[k]) < INFINITY)) w |= 127u << 8 * k;
    return w;
}
// exponent byte of a block of 4 values a lane; not finite: out of account
__device__ __forceinline__ int block_exponent(const float (&x)[4], bool in, bool& bad) {
    uint32_t t = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) t = max(t, __float_as_uint(x[k]) & 0x7fffffffu);
    t = wave_max(in ? t : 0u);
    bad = t >= 0x7f800000u;
    if (bad) {                                                   // (uniform, and rare)
        t = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) t = max(t, finite_bits(x[k]));
        t = wave_max(in ? t : 0u);
    }
    return exponent_byte(t);
}

// 16 bytes an element and some 90 instructions, 28.5 M elements in 300 tensors 82 us = 5.5 TB/s: close to where the vector units would
// bound it, hence the conversion instructions, the roots off one instruction and maxima without LDS (146 instructions an element and
// 103 us without them).
template <bool NT, bool OWN>
__global__ __launch_bounds__(256) void adamw8_kernel(float* __restrict__ p, const float* __restrict__ g, uint8_t* __restrict__ m,
                                                     uint8_t* __restrict__ r, uint8_t* __restrict__ ms, uint8_t* __restrict__ rs,
                                                     const Row* __restrict__ table, Step step) {
    const Row row = table[blockIdx.x];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), e = threadIdx.x * 4;
    const bool in = e < row.count, live = wave * 256 < row.count;        // (live: whole waves)
    if (!OWN && !live) return;
    const int first = live ? wave * 256 : 0;                     // lanes and waves past the end read a block's first elements
    const int64_t i = row.first + (in ? e : first), blk = row.block + (live ? wave : 0);
    f32x4 pv = ldv<NT>(quad(p + i));
    const f32x4 gv = ldv<NT>(quad(g + i));
    const uint32_t mc = ldv<NT>(reinterpret_cast<const uint32_t*>(m + i)), rc = ldv<NT>(reinterpret_cast<const uint32_t*>(r + i));
    const float msc = pow2((int)ms[blk] - 127), rsc = pow2((int)rs[blk] - 127);
    Coef k;
    float clip;
    uint32_t key;
    settings<OWN>(step, row.group, k, clip, key);
    if (!live) return;
    const uint32_t base = (uint32_t)i * GOLD + key;
    float mv[4], rv[4];
    uint32_t um[4], ur[4];
    decode(mv, mc);
    decode(rv, rc);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float gj = scaled(gv[j], clip), b = rv[j] * rsc;
        mv[j] = moment1(mv[j] * msc, gj, k);
        rv[j] = root<true>(moment2(b * b, gj, k));
        pv[j] = weight(pv[j], mv[j], rv[j], k);
        const uint32_t h = mix32(base + j * GOLD);
        um[j] = h & 0xffff0000u;
        ur[j] = h << 16;
    }
    bool badm, badr;
    const int em = block_exponent(mv, in, badm), er = block_exponent(rv, in, badr);
    uint32_t mw = encode(mv, pow2(127 - em), um), rw = at_least_one(encode(rv, pow2(127 - er), ur), rv);
    if (badm || badr) {
        mw = poison(mw, mv);
        rw = poison(rw, rv);
    }
    if (in) {
        stv<NT>(quad(p + i), pv);
        stv<NT>(reinterpret_cast<uint32_t*>(m + i), mw);
        stv<NT>(reinterpret_cast<uint32_t*>(r + i), rw);
    }
    if ((threadIdx.x & 63) == 0) { ms[blk] = (uint8_t)em; rs[blk] = (uint8_t)er; }
}

// fp32 moments <-> codes (root: the codes hold the square root); packing rounds to nearest
__global__ __launch_bounds__(256) void pack8_kernel(const float* __restrict__ x, uint8_t* __restrict__ code, uint8_t* __restrict__ scale,
                                                    const Row* __restrict__ table, int of_root) {
    const Row row = table[blockIdx.x];
    const int wave = threadIdx.x >> 6;
    if (wave * 256 >= row.count) return;
    const int e = threadIdx.x * 4;
    const bool in = e < row.count;
    const uint32_t half[4] = {0x80000000u, 0x80000000u, 0x80000000u, 0x80000000u};
    float xv[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const float a = in ? x[row.first + e + k] : 0.f;
        xv[k] = of_root ? root<true>(a) : a;
    }
    bool bad;
    const int eb = block_exponent(xv, in, bad);
    uint32_t w = encode(xv, pow2(127 - eb), half);
    if (of_root) w = at_least_one(w, xv);
    if (bad) w = poison(w, xv);
    if (in) *reinterpret_cast<uint32_t*>(code + row.first + e) = w;
    if ((threadIdx.x & 63) == 0) scale[row.block + wave] = (uint8_t)eb;
}

__global__ __launch_bounds__(256) void unpack8_kernel(const uint8_t* __restrict__ code, const uint8_t* __restrict__ scale,
                                                      float* __restrict__ x, const Row* __restrict__ table, int root) {
    const Row row = table[blockIdx.x];
    const int e = threadIdx.x * 4;
    if (e >= row.count) return;
    const float s = pow2((int)scale[row.block + (threadIdx.x >> 6)] - 127);
    float v[4];
    decode(v, *reinterpret_cast<const uint32_t*>(code + row.first + e));
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const float a = v[k] * s;
        x[row.first + e + k] = root ? a * a : a;
    }
}

// What a step touches, from its chunks, against the last-level cache of 256 MB.  Past the caches / through them, us (steps replayed
// from a HIP graph, three optimizers in turn): 63.6 M elements in 32 bits (1.8 GB, clipped) 306 / 392, 28.5 M (800 MB) 131 / 151, 10 M
// (280 MB) 50 / 57, 3 M (84 MB) 17.6 / 16.4; in 8 bits 28.5 M (456 MB) 79 / 86, 10 M (160 MB) 31.6 / 32.0, 3 M (48 MB) 12.9 / 12.8.
bool stream_past(int chunks, int bytes) { return (int64_t)chunks * 1024 * bytes > (256ll << 20); }

// In a small step each workgroup works out the coefficients for itself (two powers by squaring, hidden behind its loads): a launch
// less.  Itself / a launch before, us: 20 000 elements 3.4 / 4.5 in 32 bits and 4.0 / 5.1 in 8, 100 000 4.4 / 4.7 and 4.9 / 5.2, 200 000
// 5.4 / 4.9 and 6.0 / 5.3, 1 000 000 16.8 / 8.5 and 15.9 / 7.3 (the tickets queue up), and 4 us of host time in each.
bool on_its_own(int chunks) { return chunks <= 128; }

bool step_ok(const void* p, const void* g, const void* table, int chunks, const Step& s) {
    return p && g && table && chunks >= 1 && s.hyper && s.groups >= 1 && s.step && s.coef &&
           (s.part == nullptr ? s.nparts == 0 : (s.nparts >= 1 && s.norm_out != nullptr));
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
    const Step s = {hyper, groups, step, part, nparts, norm_out, 0u, coef};
    if (!step_ok(p, g, table, chunks, s) || !m || !v) return ADVMIX_EINVAL;
    hipStream_t st = (hipStream_t)stream;
    const Row* rows = reinterpret_cast<const Row*>(table);
    const dim3 grid(chunks), block(256);
    if (on_its_own(chunks)) hipLaunchKernelGGL((adamw_kernel<false, true>), grid, block, 0, st, p, g, m, v, rows, s);
    else {
        hipLaunchKernelGGL(tick_kernel, dim3(1), block, 0, st, s);
        if (stream_past(chunks, 28)) hipLaunchKernelGGL((adamw_kernel<true, false>), grid, block, 0, st, p, g, m, v, rows, s);
        else hipLaunchKernelGGL((adamw_kernel<false, false>), grid, block, 0, st, p, g, m, v, rows, s);
    }
    ADVMIX_CHECK_LAUNCH();
    return ADVMIX_OK;
}

extern "C" int advmix_adamw8(float* p, const float* g, uint8_t* m, uint8_t* r, uint8_t* m_scale, uint8_t* r_scale,
                             const int64_t* table, int chunks, const double* hyper, int groups, int64_t* step, const double* part,
                             int nparts, float* norm_out, int seed, float* coef, void* stream) {
    const Step s = {hyper, groups, step, part, nparts, norm_out, (uint32_t)seed, coef};
    if (!step_ok(p, g, table, chunks, s) || !m || !r || !m_scale || !r_scale) return ADVMIX_EINVAL;
    hipStream_t st = (hipStream_t)stream;
    const Row* rows = reinterpret_cast<const Row*>(table);
    const dim3 grid(chunks), block(256);
    if (on_its_own(chunks)) hipLaunchKernelGGL((adamw8_kernel<false, true>), grid, block, 0, st, p, g, m, r, m_scale, r_scale, rows, s);
    else {
        hipLaunchKernelGGL(tick_kernel, dim3(1), block, 0, st, s);
        if (stream_past(chunks, 16)) hipLaunchKernelGGL((adamw8_kernel<true, false>), grid, block, 0, st, p, g, m, r, m_scale, r_scale, rows, s);
        else hipLaunchKernelGGL((adamw8_kernel<false, false>), grid, block, 0, st, p, g, m, r, m_scale, r_scale, rows, s);
    }
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
