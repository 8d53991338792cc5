// Layer norm over the channels of a row (a pixel of an NHWC map, or a token), forward and backward, for fp32, bf16 and fp16
// activations with fp32 parameters:
//   y = (x - mean) * rstd * gamma + beta,  rstd = 1 / sqrt(var + eps)
//   dx = rstd * (h - mean(h) - xh * mean(h * xh)),  h = dy * gamma,  xh = (x - mean) * rstd
//   dgamma += sum over rows of dy * xh,  dbeta += sum over rows of dy
// Statistics and sums are fp32; the variance is the mean of (x - mean)^2, not E[x^2] - mean^2, so that a mean far from zero
// costs no digits.  The only rounding to fewer bits is that of y and dx to the activations' type.
//
// Bound by memory: forward reads x and writes y, backward reads x and dy and writes dx.  A row is held in registers by L lanes,
// NV 16-byte chunks each, so that every pass over it after the first is free; a wave holds 64 / L short rows at once, a long
// row is held by a workgroup of L lanes.  The backward kernel also carries its lanes' column sums of dy * xh and dy from row to
// row - gamma's and beta's gradients cost no second reading - and leaves one partial row per workgroup; ln_fold_kernel adds
// them in a fixed order.
#include "common.h"

namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
struct bf16 { uint16_t b; };
struct f16 { _Float16 v; };

// V elements of T: 16 bytes, loaded and stored at element alignment (global memory takes 16-byte accesses at any address)
template <typename T> struct Vec;
template <> struct Vec<float> {
    static constexpr int V = 4;
    typedef u32x4 Raw __attribute__((aligned(4)));
    static __device__ __forceinline__ float get(const u32x4& w, int e) { return __uint_as_float(w[e]); }
    static __device__ __forceinline__ u32x4 put(const float (&f)[4]) {
        return u32x4{__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3])};
    }
    static __device__ __forceinline__ float ld(const float* p) { return *p; }
    static __device__ __forceinline__ void st(float* p, float v) { *p = v; }
};
template <> struct Vec<bf16> {
    static constexpr int V = 8;
    typedef u32x4 Raw __attribute__((aligned(2)));
    static __device__ __forceinline__ float get(const u32x4& w, int e) {
        return __uint_as_float(e & 1 ? w[e >> 1] & 0xffff0000u : w[e >> 1] << 16);
    }
    static __device__ __forceinline__ u32x4 put(const float (&f)[8]) {
        u32x4 w;
#pragma unroll
        for (int k = 0; k < 4; ++k) w[k] = __builtin_bit_cast(uint32_t, bf16x2{(__bf16)f[2 * k], (__bf16)f[2 * k + 1]});
        return w;
    }
    static __device__ __forceinline__ float ld(const bf16* p) { return __uint_as_float((uint32_t)p->b << 16); }
    static __device__ __forceinline__ void st(bf16* p, float v) { p->b = __builtin_bit_cast(uint16_t, (__bf16)v); }
};
template <> struct Vec<f16> {
    static constexpr int V = 8;
    typedef u32x4 Raw __attribute__((aligned(2)));
    static __device__ __forceinline__ float get(const u32x4& w, int e) {
        return (float)__builtin_bit_cast(_Float16, (uint16_t)(e & 1 ? w[e >> 1] >> 16 : w[e >> 1] & 0xffffu));
    }
    static __device__ __forceinline__ u32x4 put(const float (&f)[8]) {
        u32x4 w;
#pragma unroll
        for (int k = 0; k < 4; ++k)
            w[k] = (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)f[2 * k]) |
                   ((uint32_t)__builtin_bit_cast(uint16_t, (_Float16)f[2 * k + 1]) << 16);
        return w;
    }
    static __device__ __forceinline__ float ld(const f16* p) { return (float)p->v; }
    static __device__ __forceinline__ void st(f16* p, float v) { p->v = (_Float16)v; }
};
template <typename T> __device__ __forceinline__ u32x4 load(const T* p) {
    return *reinterpret_cast<const typename Vec<T>::Raw*>(p);
}
template <typename T> __device__ __forceinline__ u32x4 load_past(const T* p) {            // past the caches
    return __builtin_nontemporal_load(reinterpret_cast<const typename Vec<T>::Raw*>(p));
}
template <typename T> __device__ __forceinline__ void store(T* p, const u32x4& w) {
    *reinterpret_cast<typename Vec<T>::Raw*>(p) = w;
}

// Sum over the L neighbouring lanes of a row, in every one of them: each step adds a permutation under which the sums so far
// are constant (lane ^ 1, lane ^ 2, mirrors of 8 and 16 lanes, the other row of 16, the other half), so no LDS is used.
template <int CTRL> __device__ __forceinline__ float dpp(float v) {
    return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), CTRL, 0xf, 0xf, true));
}
template <int L> __device__ __forceinline__ float lanes_sum(float v) {
    if (L >= 2) v += dpp<0xB1>(v);
    if (L >= 4) v += dpp<0x4E>(v);
    if (L >= 8) v += dpp<0x141>(v);
    if (L >= 16) v += dpp<0x140>(v);
    if (L >= 32) {
        const u32x2 s = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(s[0]) + __uint_as_float(s[1]);
    }
    if (L >= 64) {
        const u32x2 s = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(s[0]) + __uint_as_float(s[1]);
    }
    return v;
}
// Sum over the lanes of a wave with the same place in their rows of L lanes, in every one of them (rotations within 16 lanes
// first: what they add has a period by then).
template <int L> __device__ __forceinline__ float places_sum(float v) {
    if (L <= 8) v += dpp<0x128>(v);
    if (L <= 4) v += dpp<0x124>(v);
    if (L <= 2) v += dpp<0x122>(v);
    if (L <= 1) v += dpp<0x121>(v);
    if (L <= 16) {
        const u32x2 s = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(s[0]) + __uint_as_float(s[1]);
    }
    if (L <= 32) {
        const u32x2 s = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(s[0]) + __uint_as_float(s[1]);
    }
    return v;
}
// ... over a row held by L of the workgroup's TH lanes.  L > 64: the waves' sums meet in LDS (box: 2 * TH / 64 floats; ``flip``
// alternates its halves, so the one barrier of a sum separates the reading of the other half from its next writing)
template <int L, int TH> __device__ __forceinline__ float row_sum(float v, float* box, int& flip) {
    v = lanes_sum<L < 64 ? L : 64>(v);
    if (L > 64) {
        constexpr int W = L / 64;
        const int wave = threadIdx.x >> 6;
        float* b = box + flip * (TH / 64);
        flip ^= 1;
        if ((threadIdx.x & 63) == 0) b[wave] = v;
        __syncthreads();
        v = lanes_sum<W>(b[wave / W * W + (threadIdx.x & (W - 1))]);
    }
    return v;
}

// Where lane l of a row finds its chunk k.  With C % V != 0 the last chunk is moved back to end with the row: its elements
// before ``from`` are another lane's (read and written twice, with the same bits; summed once).  Needs C >= V.
template <int V, int L, bool TAIL> struct Place {
    int at, from;
    bool any;
    __device__ __forceinline__ Place(int k, int l, int C) {
        const int c = (k * L + l) * V;
        any = c < C;
        at = TAIL ? (c < C - V ? c : C - V) : (any ? c : 0);
        from = any ? c - at : V;
    }
    // v for an element that is this lane's, 0 for one that another lane sums; a chunk behind the row is left to the caller
    __device__ __forceinline__ float own(float v, int e) const { return !TAIL || e >= from ? v : 0.f; }
};
__device__ __forceinline__ u32x4 zero_unless(bool yes, const u32x4& w) {
    return yes ? w : u32x4{0u, 0u, 0u, 0u};
}

// V elements of gamma or beta (``none`` where there is no such tensor); one uniform branch a chunk, so that all loads are in
// flight together.
template <int V> __device__ __forceinline__ void params(float (&to)[V], const float* __restrict__ p, int at, float none) {
    typedef f32x4 Four __attribute__((aligned(4)));
    if (p) {
#pragma unroll
        for (int q = 0; q < V / 4; ++q) {
            const f32x4 f = *reinterpret_cast<const Four*>(p + at + 4 * q);
#pragma unroll
            for (int e = 0; e < 4; ++e) to[4 * q + e] = f[e];
        }
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e) to[e] = none;
    }
}

constexpr int threads_of(int L) { return L > 256 ? L : 256; }

// (Times here and below: launches replayed from a HIP graph, three sets of data in turn, each with outputs of its own.)
// One reading, one writing: 12289 x 2048 fp32 38 us = 5.2 TB/s (33 us = 6.1 TB/s where y is the memory of the call before), 16384 x
// 4096 bf16 53 us = 5.1 TB/s (46 us), 32 x 64 x 48 pixels of 32 channels 6.1 us.  Workgroups walk the rows, so that gamma and beta
// are read once; without the next row on its way the second case's 46 us are 66.
template <typename T, int L, int NV, bool TAIL>
__global__ __launch_bounds__(threads_of(L)) void ln_fwd_kernel(const T* __restrict__ x, int64_t ldx, const float* __restrict__ gamma,
                                                               const float* __restrict__ beta, T* __restrict__ y,
                                                               float* __restrict__ mean, float* __restrict__ rstd, int64_t rows, int C,
                                                               float eps) {
    constexpr int V = Vec<T>::V, TH = threads_of(L), R = TH / L;
    __shared__ float box[2 * TH / 64];
    const int l = threadIdx.x % L;
    int flip = 0;
    const float n = (float)C;                                    // (a division: the mean of equal values is that value)
    const int64_t step = (int64_t)gridDim.x * R;
    int64_t r = (int64_t)blockIdx.x * R + threadIdx.x / L;
    u32x4 next[NV];                                              // the next row is on its way while this one is worked on
    const auto fetch = [&](int64_t row) {
        const T* xr = x + (row < rows ? row : rows - 1) * ldx;   // (a lane without a row reads the last one)
#pragma unroll
        for (int k = 0; k < NV; ++k) next[k] = load(xr + Place<V, L, TAIL>(k, l, C).at);
    };
    fetch(r);
    float gm[NV][V], bt[NV][V];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int at = Place<V, L, TAIL>(k, l, C).at;
        params<V>(gm[k], gamma, at, 1.f);
        params<V>(bt[k], beta, at, 0.f);
    }
    for (int64_t r0 = (int64_t)blockIdx.x * R; r0 < rows; r0 += step, r += step) {
        const bool in = r < rows;
        u32x4 w[NV];
#pragma unroll
        for (int k = 0; k < NV; ++k) w[k] = next[k];
        if (r0 + step < rows) fetch(r + step);
        float s = 0.f;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const Place<V, L, TAIL> at(k, l, C);
            float part = 0.f;
#pragma unroll
            for (int e = 0; e < V; ++e) part += at.own(Vec<T>::get(w[k], e), e);
            s += at.any ? part : 0.f;
        }
        const float mu = row_sum<L, TH>(s, box, flip) / n;
        float q = 0.f;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const Place<V, L, TAIL> at(k, l, C);
            float part = 0.f;
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float d = at.own(Vec<T>::get(w[k], e) - mu, e);
                part = fmaf(d, d, part);
            }
            q += at.any ? part : 0.f;
        }
        const float is = 1.f / sqrtf(row_sum<L, TH>(q, box, flip) / n + eps);
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const Place<V, L, TAIL> at(k, l, C);
            float o[V];
#pragma unroll
            for (int e = 0; e < V; ++e) o[e] = fmaf((Vec<T>::get(w[k], e) - mu) * is, gm[k][e], bt[k][e]);
            if (in && at.any) store(y + r * C + at.at, Vec<T>::put(o));
        }
        if (mean && in && l == 0) { mean[r] = mu; rstd[r] = is; }
    }
}

// to[c] += v or = v
__device__ __forceinline__ void give(float* to, int64_t c, float v, int add) {
    if (!to) return;
    if (add) atomicAdd(to + c, v);                               // (one per sum and launch: see ln_fold_kernel)
    else to[c] = v;
}

// part[workgroup][0][c] = sum of dy * xh, [1][c] = sum of dy over the workgroup's rows; a launch of one workgroup gives its sums
// to dgamma and dbeta itself (part NULL; not one of long rows, whose lanes would write them one element at a time).
// Two readings, one writing, with the folding launch: 16384 x 4096 bf16 76 us = 5.3 TB/s, 100000 x 256 fp32 58 us = 5.3 TB/s, the same
// without the sums 73 and 57 us.  Vector work matters: masks per element instead of per chunk are 8 us more in the first case.
// PAST: x is read past the caches (dy is what another kernel has just left there).
template <typename T, int L, int NV, bool TAIL, bool PAST>
__global__ __launch_bounds__(L > 512 ? L : 512) void ln_bwd_kernel(const T* __restrict__ dy, int64_t lddy, const T* __restrict__ x,
                                                                 int64_t ldx, const float* __restrict__ gamma,
                                                                 const float* __restrict__ mean, const float* __restrict__ rstd,
                                                                 T* __restrict__ dx, float* dgamma, float* dbeta,
                                                                 float* __restrict__ part, int add,
                                                                 int64_t rows, int C) {
    constexpr int V = Vec<T>::V, TH = L > 512 ? L : 512, R = TH / L, W = TH / 64;
    extern __shared__ float lds[];                               // row sums' box, then the workgroup's column sums [R waves][C]
    const int l = threadIdx.x % L;
    int flip = 0;
    // 1024 lanes may have 128 registers each: with 16 elements a lane there is no room for the next row, and gamma is read again
    // (from the L2) with every row
    constexpr bool ROOM = L < 1024 || NV * V < 16;
    const float n = (float)C;
    const int64_t step = (int64_t)gridDim.x * R;
    int64_t r = (int64_t)blockIdx.x * R + threadIdx.x / L;
    u32x4 nw[NV], ng[NV];                                        // the next row is on its way while this one is worked on
    float nmu, nis;
    const auto fetch = [&](int64_t row) {
        const int64_t rr = row < rows ? row : rows - 1;
        const T *xr = x + rr * ldx, *gr = dy + rr * lddy;
        nmu = mean[rr];
        nis = rstd[rr];
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int at = Place<V, L, TAIL>(k, l, C).at;
            nw[k] = PAST ? load_past(xr + at) : load(xr + at);
            ng[k] = load(gr + at);
        }
    };
    if (ROOM) fetch(r);
    float gm[NV][V], dg[NV][V], db[NV][V];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
#pragma unroll
        for (int e = 0; e < V; ++e) dg[k][e] = db[k][e] = 0.f;
        if (ROOM) params<V>(gm[k], gamma, Place<V, L, TAIL>(k, l, C).at, 1.f);
    }
    for (int64_t r0 = (int64_t)blockIdx.x * R; r0 < rows; r0 += step, r += step) {
        const bool in = r < rows;
        if (!ROOM) fetch(r);
        // without a row: xh = 0 and dy = 0, whatever the last row holds; behind the row (a chunk of none): dy = 0
        const float mu = in ? nmu : 0.f, is = in ? nis : 0.f;
        u32x4 w[NV], g[NV];
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            w[k] = zero_unless(in, nw[k]);
            g[k] = zero_unless(in && Place<V, L, TAIL>(k, l, C).any, ng[k]);
        }
        if (ROOM && r0 + step < rows) fetch(r + step);
        float a = 0.f, b = 0.f;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const Place<V, L, TAIL> at(k, l, C);
            if (!ROOM) params<V>(gm[k], gamma, at.at, 1.f);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float xh = (Vec<T>::get(w[k], e) - mu) * is;
                const float d = at.own(Vec<T>::get(g[k], e), e), h = d * gm[k][e];
                a += h;
                b = fmaf(h, xh, b);
                dg[k][e] = fmaf(d, xh, dg[k][e]);                // (of elements that are another lane's, never used)
                db[k][e] += d;
            }
        }
        a = row_sum<L, TH>(a, lds, flip) / n * is;
        b = row_sum<L, TH>(b, lds, flip) / n * is;
        if (dx) {
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                const Place<V, L, TAIL> at(k, l, C);
                float o[V];
                if (!ROOM) params<V>(gm[k], gamma, at.at, 1.f);
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const float xh = (Vec<T>::get(w[k], e) - mu) * is;
                    o[e] = fmaf(Vec<T>::get(g[k], e) * gm[k][e], is, -fmaf(xh, b, a));
                }
                if (in && at.any) store(dx + r * C + at.at, Vec<T>::put(o));
            }
        }
    }
    if (!dgamma && !dbeta) return;
    if (R == 1) {                                                // one row at a time: a lane has its columns to itself (part is there)
        typedef f32x4 Four __attribute__((aligned(4)));
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            float* row = part + ((int64_t)blockIdx.x * 2 + which) * C;
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                const Place<V, L, TAIL> at(k, l, C);
                const float(&v)[V] = which ? db[k] : dg[k];
                if (at.from == 0) {
#pragma unroll
                    for (int q = 0; q < V; q += 4)
                        *reinterpret_cast<Four*>(row + at.at + q) = f32x4{v[q], v[q + 1], v[q + 2], v[q + 3]};
                } else {
#pragma unroll
                    for (int e = 0; e < V; ++e)
                        if (e >= at.from) row[at.at + e] = v[e];       // (from = V where the chunk lies behind the row)
                }
            }
        }
        return;
    }
    // the rows of a wave are added across its lanes, those of different waves in LDS; first dg, then db
    constexpr int G = R < W ? R : W;
    const int wide = TAIL ? C + (C >> 3) + 1 : C;                // (element by element, every ninth word is left out: a lane's next
#pragma unroll                                                   //  eight columns then start in another bank)
    for (int which = 0; which < 2; ++which) {
        const float(&s)[NV][V] = which ? db : dg;
        __syncthreads();
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const Place<V, L, TAIL> at(k, l, C);
            float v[V];
#pragma unroll
            for (int e = 0; e < V; ++e) v[e] = places_sum<L>(s[k][e]);
            const bool mine = L >= 64 || (threadIdx.x & 63) < L;
            float* to = lds + (L >= 64 ? threadIdx.x / L : threadIdx.x >> 6) * wide;
            if (!TAIL) {                                         // C is a multiple of V: 16-byte writes
                if (mine && at.any)
#pragma unroll
                    for (int q = 0; q < V; q += 4)
                        *reinterpret_cast<f32x4*>(to + at.at + q) = f32x4{v[q], v[q + 1], v[q + 2], v[q + 3]};
            } else {
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const int c = at.at + e;
                    if (mine && e >= at.from) to[c + (c >> 3)] = v[e];
                }
            }
        }
        __syncthreads();
        float* to = which ? dbeta : dgamma;
        for (int c = threadIdx.x; c < C; c += TH) {
            const int j = TAIL ? c + (c >> 3) : c;
            float v = 0.f;
#pragma unroll
            for (int i = 0; i < G; ++i) v += lds[i * wide + j];
            if (part) part[((int64_t)blockIdx.x * 2 + which) * C + c] = v;
            else give(to, c, v, add & (1 << which));
        }
    }
}

// The workgroups' partial sums in a fixed order: 16 columns x 64 slices of the partial rows per workgroup, so that a thread has at
// most eight loads, all in flight (2.5 - 3.8 us, a launch's own time; 5 us for 4096 columns).  With ``add`` ONE atomic addition per
// sum, so that two launches that add to one gradient (or one launch whose dgamma and dbeta are one) lose neither's part; a launch
// that stores is for a gradient that no other one touches before it has run.
constexpr int FOLD = 16;
__global__ __launch_bounds__(1024) void ln_fold_kernel(const float* __restrict__ part, int parts, float* dgamma, float* dbeta,
                                                       int add, int C) {
    constexpr int S = 1024 / FOLD;
    __shared__ float box[FOLD][S + 1];
    const int j = threadIdx.x % FOLD, s = threadIdx.x / FOLD;
    const int c = blockIdx.x * FOLD + j, which = blockIdx.y;
    const float* at = part + (int64_t)which * C + (c < C ? c : 0);
    float v[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
        const int i = s + u * S;
        v[u] = at[(int64_t)(i < parts ? i : 0) * 2 * C];
        v[u] = i < parts ? v[u] : 0.f;
    }
    box[j][s] = ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
    __syncthreads();
    const int wave = threadIdx.x >> 6;                           // a wave a column
    const float sum = lanes_sum<64>(box[wave][threadIdx.x & 63]);
    const int col = blockIdx.x * FOLD + wave;
    if ((threadIdx.x & 63) == 0 && col < C) give(which ? dbeta : dgamma, col, sum, add & (1 << which));
}

// ---- rows that no workgroup holds (or fewer channels than a chunk): a workgroup walks the row, element by element -------
// Built to be right, not fast: below a chunk at most seven lanes of a wave have an element and the column kernel as many of its 256
// threads (70001 x 3 fp32 17 us forward and 48 backward, 100000 x 7 bf16 25 and 85, where memory would take 1).
template <typename T, int TH>
__global__ __launch_bounds__(TH) void ln_fwd_walk_kernel(const T* __restrict__ x, int64_t ldx, const float* __restrict__ gamma,
                                                         const float* __restrict__ beta, T* __restrict__ y, float* __restrict__ mean,
                                                         float* __restrict__ rstd, int64_t rows, int C, float eps) {
    __shared__ float box[2 * TH / 64];
    int flip = 0;
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
        const T* xr = x + r * ldx;
        float s = 0.f, q = 0.f;
        for (int c = threadIdx.x; c < C; c += TH) s += Vec<T>::ld(xr + c);
        const float mu = row_sum<TH, TH>(s, box, flip) / C;
        for (int c = threadIdx.x; c < C; c += TH) {
            const float d = Vec<T>::ld(xr + c) - mu;
            q = fmaf(d, d, q);
        }
        const float is = 1.f / sqrtf(row_sum<TH, TH>(q, box, flip) / C + eps);
        for (int c = threadIdx.x; c < C; c += TH)
            Vec<T>::st(y + r * C + c, fmaf((Vec<T>::ld(xr + c) - mu) * is, gamma ? gamma[c] : 1.f, beta ? beta[c] : 0.f));
        if (mean && threadIdx.x == 0) { mean[r] = mu; rstd[r] = is; }
    }
}

// A product rounded by itself: the same number where it is summed and where the mean is taken off it, so that one channel's dx is 0.
__device__ __forceinline__ float rounded(float a, float b) {
#pragma clang fp contract(off)
    return a * b;
}
template <typename T, int TH>
__global__ __launch_bounds__(TH) void ln_dx_walk_kernel(const T* __restrict__ dy, int64_t lddy, const T* __restrict__ x, int64_t ldx,
                                                        const float* __restrict__ gamma, const float* __restrict__ mean,
                                                        const float* __restrict__ rstd, T* __restrict__ dx, int64_t rows, int C) {
    __shared__ float box[2 * TH / 64];
    int flip = 0;
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
        const T *xr = x + r * ldx, *gr = dy + r * lddy;
        const float mu = mean[r], is = rstd[r];
        float a = 0.f, b = 0.f;
        for (int c = threadIdx.x; c < C; c += TH) {
            const float h = rounded(Vec<T>::ld(gr + c), gamma ? gamma[c] : 1.f);
            a += h;
            b += h * ((Vec<T>::ld(xr + c) - mu) * is);
        }
        a = row_sum<TH, TH>(a, box, flip) / C;
        b = row_sum<TH, TH>(b, box, flip) / C;
        for (int c = threadIdx.x; c < C; c += TH) {
            const float h = rounded(Vec<T>::ld(gr + c), gamma ? gamma[c] : 1.f);
            Vec<T>::st(dx + r * C + c, is * (h - a - (Vec<T>::ld(xr + c) - mu) * is * b));
        }
    }
}

template <typename T>
__global__ __launch_bounds__(256) void ln_columns_kernel(const T* __restrict__ dy, int64_t lddy, const T* __restrict__ x, int64_t ldx,
                                                         const float* __restrict__ mean, const float* __restrict__ rstd,
                                                         float* __restrict__ part, int64_t rows, int C) {
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= C) return;
    float dg = 0.f, db = 0.f;
    for (int64_t r = blockIdx.y; r < rows; r += gridDim.y) {
        const float g = Vec<T>::ld(dy + r * lddy + c);
        dg = fmaf(g, (Vec<T>::ld(x + r * ldx + c) - mean[r]) * rstd[r], dg);
        db += g;
    }
    part[(blockIdx.y * 2ll) * C + c] = dg;
    part[(blockIdx.y * 2ll + 1) * C + c] = db;
}

// ---- which kernel holds a row ------------------------------------------------------------------------------------------
// chunks of 16 bytes per row -> (L lanes, NV chunks a lane); {0, 0}: no workgroup holds it
struct Hold { int L, NV; };
Hold hold_of(int C, int V) {
    if (C < V) return {0, 0};
    const int n = (C + V - 1) / V, most = V == 4 ? 4 : 2;        // at most 16 elements a lane: the backward kernel keeps five values of each
    for (int L = 1; L <= 64; L *= 2)
        if (n <= L) return {L, 1};
    for (int NV = 2; NV <= most; ++NV)
        if (n <= 64 * NV) return {64, NV};
    for (int NV = 1; NV <= most; ++NV)
        if (n <= 256 * NV) return {256, NV};
    for (int NV = 1; NV <= most; NV *= 2)
        if (n <= 1024 * NV) return {1024, NV};
    return {0, 0};
}

// Workgroups of the backward kernel where it sums columns: as many as the chip holds at once (with 16 elements a lane one of
// 512 lanes per CU, two otherwise; a long row's 1024 lanes one), each with the same number of rows, give or take one.
int parts_of(int64_t rows, int C, int V) {
    const Hold h = hold_of(C, V);
    if (h.L == 0) return (int)(rows < 256 ? rows : 256);         // column kernel: slices of the rows
    const int R = (h.L > 512 ? h.L : 512) / h.L;
    const int64_t units = (rows + R - 1) / R, most = h.L == 1024 || h.NV * V >= 16 ? 256 : 512;
    if (R > 1 && units <= 2) return 1;                           // (one workgroup, no folding: 16 x 768 bf16 5.1 us, 1 us more with two)
    const int64_t each = (units + most - 1) / most;
    return (int)((units + each - 1) / each);
}

// what hold_of returns: for every type, for fp32, for 16 bits
#define HOLDS(CASE)                                                                                               \
    CASE(1, 1) CASE(2, 1) CASE(4, 1) CASE(8, 1) CASE(16, 1) CASE(32, 1) CASE(64, 1) CASE(64, 2) CASE(256, 2) CASE(1024, 2)
#define HOLDS_F32(CASE) CASE(64, 3) CASE(64, 4) CASE(256, 3) CASE(256, 4) CASE(1024, 4)
#define HOLDS_16(CASE) CASE(256, 1) CASE(1024, 1)

template <typename T>
int fwd(const void* x_, int64_t ldx, const float* gamma, const float* beta, void* y_, float* mean, float* rstd, int64_t rows, int C,
        float eps, hipStream_t st) {
    constexpr int V = Vec<T>::V;
    const T* x = (const T*)x_;
    T* y = (T*)y_;
    const Hold h = hold_of(C, V);
    const int R = h.L ? threads_of(h.L) / h.L : 1;
    int64_t grid = (rows + R - 1) / R;
    const int64_t cap = h.L > 256 ? 512 : 2048;                  // what 256 CUs hold at once, or twice that
    if (grid > cap) grid = cap;
    const dim3 g((unsigned)grid);
#define FWD(L_, NV_)                                                                                                            \
    if (h.L == L_ && h.NV == NV_) {                                                                                             \
        constexpr bool ODD = L_ > 1;                             /* (one lane holds one whole chunk or nothing) */              \
        if (ODD && C % V) hipLaunchKernelGGL((ln_fwd_kernel<T, L_, NV_, ODD>), g, dim3(threads_of(L_)), 0, st, x, ldx, gamma,   \
                                             beta, y, mean, rstd, rows, C, eps);                                                \
        else hipLaunchKernelGGL((ln_fwd_kernel<T, L_, NV_, false>), g, dim3(threads_of(L_)), 0, st, x, ldx, gamma, beta, y, mean, \
                                rstd, rows, C, eps);                                                                            \
    }
    HOLDS(FWD)
    if constexpr (V == 4) { HOLDS_F32(FWD) } else { HOLDS_16(FWD) }
#undef FWD
    if (h.L == 0) {
        if (C < V) hipLaunchKernelGGL((ln_fwd_walk_kernel<T, 64>), dim3((unsigned)(rows < 8192 ? rows : 8192)), dim3(64), 0, st, x, ldx, gamma, beta, y, mean, rstd, rows, C, eps);
        else hipLaunchKernelGGL((ln_fwd_walk_kernel<T, 1024>), dim3((unsigned)(rows < 512 ? rows : 512)), dim3(1024), 0, st, x, ldx, gamma, beta, y, mean, rstd, rows, C, eps);
    }
    ADVMIX_CHECK_LAUNCH();
    return ADVMIX_OK;
}

template <typename T>
int bwd(const void* dy_, int64_t lddy, const void* x_, int64_t ldx, const float* gamma, const float* mean, const float* rstd, void* dx_,
        float* dgamma, float* dbeta, float* part, int add, int64_t rows, int C, hipStream_t st) {
    constexpr int V = Vec<T>::V;
    const T *x = (const T*)x_, *dy = (const T*)dy_;
    T* dx = (T*)dx_;
    const Hold h = hold_of(C, V);
    const int parts = parts_of(rows, C, V);
    const bool sums = dgamma || dbeta;
    if (h.L) {
        const int TH = h.L > 512 ? h.L : 512, R = TH / h.L, W = TH / 64;
        const int64_t need = (rows + R - 1) / R;
        const dim3 g((unsigned)(sums ? parts : (need < 2048 ? need : 2048)));
        const size_t lds = sums && R > 1 ? sizeof(float) * ((R < W ? R : W) * (size_t)(C % V ? C + (C >> 3) + 1 : C)) : 0, box = sizeof(float) * 2 * W;
        float* pp = parts > 1 || R == 1 ? part : nullptr;
        // x, dy and dx against the last-level cache of 256 MB.  x read past the caches / through them, us, alone and with the forward
        // pass before it: 30000 x 1024 fp32 (369 MB) 69 / 72 and 109 / 112, 16384 x 4096 bf16 (403 MB) 76 / 79 and 125 / 129, 100000 x
        // 256 fp32 (307 MB) 58 / 61 and 96 / 93; 6144 x 768 bf16 (28 MB) 11.3 / 10.8 and 17.1 / 16.5.  With dy past them too the pass
        // behind a forward pass loses 6 - 12 %.  (Odd widths keep to the caches: neighbouring rows share lines.)
        const bool past = rows * C * (int64_t)sizeof(T) * 3 > (256ll << 20);
#define BWD(L_, NV_)                                                                                                             \
    if (h.L == L_ && h.NV == NV_) {                                                                                              \
        constexpr bool ODD = L_ > 1;                                                                                             \
        if (ODD && C % V) hipLaunchKernelGGL((ln_bwd_kernel<T, L_, NV_, ODD, false>), g, dim3(TH), lds > box ? lds : box, st, dy, lddy, x, ldx, \
                                             gamma, mean, rstd, dx, dgamma, dbeta, pp, add, rows, C);                            \
        else if (past) hipLaunchKernelGGL((ln_bwd_kernel<T, L_, NV_, false, true>), g, dim3(TH), lds > box ? lds : box, st, dy, lddy, x, \
                                          ldx, gamma, mean, rstd, dx, dgamma, dbeta, pp, add, rows, C);                          \
        else hipLaunchKernelGGL((ln_bwd_kernel<T, L_, NV_, false, false>), g, dim3(TH), lds > box ? lds : box, st, dy, lddy, x, ldx, \
                                gamma, mean, rstd, dx, dgamma, dbeta, pp, add, rows, C);                                         \
    }
        HOLDS(BWD)
        if constexpr (V == 4) { HOLDS_F32(BWD) } else { HOLDS_16(BWD) }
#undef BWD
        if (!sums || !pp) { ADVMIX_CHECK_LAUNCH(); return ADVMIX_OK; }
    } else {
        if (dx) {
            if (C < V) hipLaunchKernelGGL((ln_dx_walk_kernel<T, 64>), dim3((unsigned)(rows < 8192 ? rows : 8192)), dim3(64), 0, st, dy, lddy, x, ldx, gamma, mean, rstd, dx, rows, C);
            else hipLaunchKernelGGL((ln_dx_walk_kernel<T, 1024>), dim3((unsigned)(rows < 512 ? rows : 512)), dim3(1024), 0, st, dy, lddy, x, ldx, gamma, mean, rstd, dx, rows, C);
        }
        if (sums)
            hipLaunchKernelGGL((ln_columns_kernel<T>), dim3(cdiv(C, 256), parts), dim3(256), 0, st, dy, lddy, x, ldx, mean, rstd, part, rows, C);
    }
    if (sums) hipLaunchKernelGGL(ln_fold_kernel, dim3(cdiv(C, FOLD), 2), dim3(1024), 0, st, part, parts, dgamma, dbeta, add, C);
    ADVMIX_CHECK_LAUNCH();
    return ADVMIX_OK;
}

bool sizes_ok(int64_t rows, int C, int dtype) {
    return rows >= 1 && C >= 1 && C <= (1 << 30) && dtype >= ADVMIX_F32 && dtype <= ADVMIX_F16 && rows <= INT64_MAX / 4 / C;
}

}  // namespace

extern "C" int advmix_layer_norm_parts(int64_t rows, int C, int dtype) {
    if (!sizes_ok(rows, C, dtype)) return 0;
    return parts_of(rows, C, dtype == ADVMIX_F32 ? 4 : 8);
}

extern "C" int advmix_layer_norm_fwd(const void* x, int64_t ldx, const float* gamma, const float* beta, void* y, float* mean,
                                     float* rstd, int64_t rows, int C, int dtype, float eps, void* stream) {
    if (!x || !y || ldx < 0 || (mean == nullptr) != (rstd == nullptr) || !(eps >= 0.f) || !sizes_ok(rows, C, dtype))
        return ADVMIX_EINVAL;
    hipStream_t st = (hipStream_t)stream;
    if (dtype == ADVMIX_F32) return fwd<float>(x, ldx, gamma, beta, y, mean, rstd, rows, C, eps, st);
    if (dtype == ADVMIX_BF16) return fwd<bf16>(x, ldx, gamma, beta, y, mean, rstd, rows, C, eps, st);
    return fwd<f16>(x, ldx, gamma, beta, y, mean, rstd, rows, C, eps, st);
}

extern "C" int advmix_layer_norm_bwd(const void* dy, int64_t lddy, const void* x, int64_t ldx, const float* gamma, const float* mean,
                                     const float* rstd, void* dx, float* dgamma, float* dbeta, float* part, int add, int64_t rows, int C,
                                     int dtype, void* stream) {
    if (!dy || !x || !mean || !rstd || ldx < 0 || lddy < 0 || !sizes_ok(rows, C, dtype)) return ADVMIX_EINVAL;
    if ((dgamma || dbeta) && !part) return ADVMIX_EINVAL;
    if (dgamma && dgamma == dbeta && (add & 3) != 3) return ADVMIX_EINVAL;       // (two sums in one place can only be added)
    if (!dx && !dgamma && !dbeta) return ADVMIX_OK;
    hipStream_t st = (hipStream_t)stream;
    if (dtype == ADVMIX_F32) return bwd<float>(dy, lddy, x, ldx, gamma, mean, rstd, dx, dgamma, dbeta, part, add, rows, C, st);
    if (dtype == ADVMIX_BF16) return bwd<bf16>(dy, lddy, x, ldx, gamma, mean, rstd, dx, dgamma, dbeta, part, add, rows, C, st);
    return bwd<f16>(dy, lddy, x, ldx, gamma, mean, rstd, dx, dgamma, dbeta, part, add, rows, C, st);
}
