// Attention with a sliding window and first tokens that stay visible (sinks), forward, backward and the
// single-token form over a cache (gfx950).
//
//   visible(i, j), i, j < n:   causal         j <= i and (i - j < window or j < sinks)
//                              bidirectional  |i - j| < window or j < sinks or i < sinks
//   o_i = sum_j p_ij v_j,  p_ij = exp(scale q_i.k_j - lse_i) over the visible j;  a row that sees nothing gives 0
//   dV = P^T dO;  dS = P * (dO V^T - delta), delta_i = dO_i.o_i;  dQ = scale dS K;  dK = scale dS^T Q
//
// Every product is a 32 x 32 MFMA tile.  The operand that a wave keeps (its 32 queries, or its 32 keys in the dK / dV
// kernel) sits on the MFMA column index, lane & 31, so that softmax statistics of a query are one number per lane and
// the accumulators of the first product are, as they stand, the B operand of the second: accumulator register
// r = 4 b + e of lane half h holds tile row 8 b + 4 h + e, and the second product's left operand is read from the LDS
// tile in that same order of rows.  Rows behind a sequence's length are staged as zeros, whatever memory holds there:
// a probability of zero times a NaN would be a NaN.
#include <initializer_list>

#include "common.h"

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr float LOG2E = 1.4426950408889634f;
constexpr int TQ = 128;                       // rows of a workgroup: four waves of 32

struct Slide {
    const void* q; const void* k; const void* v; void* o; float* o32; float* lse; const int* lengths;
    const void* d_o; float* delta; void* dq; void* dk; void* dv;
    int B, N, Hq, Hkv, G;
    long q_b, q_n, q_h, k_b, k_n, k_h, v_b, v_n, v_h, do_b, do_n, do_h, dq_b, dq_n, dq_h, dk_b, dk_n, dk_h, dv_b, dv_n, dv_h;
    int window, sinks;
    float scale;
};

// ----------------------------------------------------------------------------- which pairs are visible
template <bool CAUSAL> __device__ __forceinline__ bool visible(int i, int j, int n, int w, int f) {
    if (i >= n || j >= n) return false;
    if constexpr (CAUSAL) return j <= i && (i - j < w || j < f);
    const int d = i - j;
    return (d < w && -d < w) || j < f || i < f;
}
// Of the rectangle [ia, ib] x [ja, jb]: 0 nothing is visible, 2 everything is, 1 look at each pair.
template <bool CAUSAL> __device__ __forceinline__ int coverage(int ia, int ib, int ja, int jb, int n, int w, int f) {
    if (ia >= n || ja >= n) return 0;
    if constexpr (CAUSAL) {
        if (ja > ib || (ia - jb >= w && ja >= f)) return 0;
        return ib < n && jb < n && jb <= ia && (ib - ja < w || jb < f) ? 2 : 1;
    } else {
        if ((ia - jb >= w || ja - ib >= w) && ja >= f && ia >= f) return 0;
        return ib < n && jb < n && ((ib - ja < w && jb - ia < w) || jb < f || ib < f) ? 2 : 1;
    }
}
// The tiles of `T` rows of the other axis that rows [a, b] of this one can touch: [0, first) and [lo, hi).
struct Tiles { int first, lo, hi; __device__ __forceinline__ int count() const { return first + (hi > lo ? hi - lo : 0); }
               __device__ __forceinline__ int at(int t) const { return t < first ? t : lo + t - first; } };
__device__ __forceinline__ Tiles tiles_of(int lo, int hi, int first, int n, int T) {     // rows [lo, hi] and [0, first)
    Tiles t;
    first = first < n ? first : n;
    t.first = (first + T - 1) / T;
    lo = lo > 0 ? lo : 0;
    hi = hi < n - 1 ? hi : n - 1;
    t.lo = lo / T;
    t.lo = t.lo > t.first ? t.lo : t.first;
    t.hi = hi >= lo ? hi / T + 1 : 0;
    return t;
}
template <bool CAUSAL> __device__ __forceinline__ Tiles key_tiles(int qa, int qb, int n, int w, int f, int T) {
    if (qa >= n) return Tiles{0, 0, 0};
    qb = qb < n ? qb : n - 1;
    if constexpr (CAUSAL) {
        const int first = f < qb + 1 ? f : qb + 1;
        return tiles_of(qa - w + 1, w > 0 ? qb : -1, first, n, T);
    }
    if (qa < f) return tiles_of(0, n - 1, 0, n, T);
    return tiles_of(qa - w + 1, w > 0 ? qb + w - 1 : -1, f, n, T);
}
template <bool CAUSAL> __device__ __forceinline__ Tiles query_tiles(int ka, int kb, int n, int w, int f, int T) {
    if (ka >= n) return Tiles{0, 0, 0};
    kb = kb < n ? kb : n - 1;
    if constexpr (CAUSAL) return tiles_of(ka, ka < f ? n - 1 : (w > 0 ? kb + w - 1 : -1), 0, n, T);
    if (ka < f) return tiles_of(0, n - 1, 0, n, T);
    return tiles_of(ka - w + 1, w > 0 ? kb + w - 1 : -1, f, n, T);
}

// ----------------------------------------------------------------------------- operands
template <typename T, int DH> struct Shape {
    static constexpr int ROW = DH * (int)sizeof(T) + 16;          // bytes of an LDS tile row: 16 of padding
    static constexpr int CHUNKS = DH * (int)sizeof(T) / 16;
    static constexpr int KT = sizeof(T) == 2 ? 64 : 32;           // rows of a staged tile
};
// What a wave keeps of its 32 rows: column lane & 31, half h of the reduction.
template <typename T, int DH> struct Kept;
template <int DH> struct Kept<bf16_t, DH> {
    bf16x8 f[DH / 16];
    __device__ __forceinline__ void load(const bf16_t* row, int h, bool ok) {
#pragma unroll
        for (int c = 0; c < DH / 16; ++c) {
            u32x4 z = {0, 0, 0, 0};
            if (ok) z = *reinterpret_cast<const u32x4*>(row + 16 * c + 8 * h);
            f[c] = __builtin_bit_cast(bf16x8, z);
        }
    }
};
template <int DH> struct Kept<float, DH> {
    float f[DH / 2];
    __device__ __forceinline__ void load(const float* row, int h, bool ok) {
#pragma unroll
        for (int t = 0; t < DH / 8; ++t) {
            f32x4 z = {0.f, 0.f, 0.f, 0.f};
            if (ok) z = *reinterpret_cast<const f32x4*>(row + h * (DH / 2) + 4 * t);
#pragma unroll
            for (int i = 0; i < 4; ++i) f[4 * t + i] = z[i];
        }
    }
};
// 32 tile rows from r0 times the kept rows, over the head: C[row][column].
template <int DH> __device__ __forceinline__ f32x16 product(const char* tile, int r0, const Kept<bf16_t, DH>& kept, int lane) {
    f32x16 acc = {};
    const char* a = tile + (r0 + (lane & 31)) * Shape<bf16_t, DH>::ROW + (lane >> 5) * 16;
#pragma unroll
    for (int c = 0; c < DH / 16; ++c)
        acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(*reinterpret_cast<const bf16x8*>(a + 32 * c), kept.f[c], acc, 0, 0, 0);
    return acc;
}
template <int DH> __device__ __forceinline__ f32x16 product(const char* tile, int r0, const Kept<float, DH>& kept, int lane) {
    f32x16 acc = {};
    const char* a = tile + (r0 + (lane & 31)) * Shape<float, DH>::ROW + (lane >> 5) * (DH * 2);
#pragma unroll
    for (int t = 0; t < DH / 8; ++t) {
        const f32x4 x = *reinterpret_cast<const f32x4*>(a + 16 * t);
#pragma unroll
        for (int i = 0; i < 4; ++i) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(x[i], kept.f[4 * t + i], acc, 0, 0, 0);
    }
    return acc;
}
// acc[d][column] += sum over 32 tile rows from r0 of tile[row][d] * w[row][column]; w as a product left it.  In bf16
// the weights are rounded to the operand type here: 2^-9 of each, independent, and the sums stay in 32 bits.
template <int DH> __device__ __forceinline__ void gather(f32x16* acc, const char* tile, int r0, const f32x16& w, int lane, bf16_t) {
    const int l15 = lane & 15, g = lane >> 4;
    bf16x8 b[2];
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int e = 0; e < 8; ++e) b[c][e] = (bf16_t)w[8 * c + e];
    const char* a = tile + (r0 + 4 * (g >> 1) + (l15 >> 2)) * Shape<bf16_t, DH>::ROW + (16 * (g & 1) + 4 * (l15 & 3)) * 2;
#pragma unroll
    for (int d = 0; d < DH / 32; ++d) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const char* p = a + 16 * c * Shape<bf16_t, DH>::ROW + 64 * d;
            const bf16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((VITK_LDS bf16x4*)(p));
            const bf16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((VITK_LDS bf16x4*)(p + 8 * Shape<bf16_t, DH>::ROW));
            acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(bf16x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]},
                                                             b[c], acc[d], 0, 0, 0);
        }
    }
}
template <int DH> __device__ __forceinline__ void gather(f32x16* acc, const char* tile, int r0, const f32x16& w, int lane, float) {
    const char* a = tile + (r0 + 4 * (lane >> 5)) * Shape<float, DH>::ROW + (lane & 31) * 4;
#pragma unroll
    for (int d = 0; d < DH / 32; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r)
            acc[d] = __builtin_amdgcn_mfma_f32_32x32x2f32(
                *reinterpret_cast<const float*>(a + (8 * (r >> 2) + (r & 3)) * Shape<float, DH>::ROW + 128 * d), w[r], acc[d], 0, 0, 0);
}
// Rows [r0, r0 + KT) of a matrix into an LDS tile; rows from `end` on are zeros.
template <typename T, int DH, int NT> __device__ __forceinline__ void stage(char* tile, const T* base, long ld, int r0, int end, int tid) {
    constexpr int C = Shape<T, DH>::CHUNKS, ROW = Shape<T, DH>::ROW;
#pragma unroll
    for (int i = 0; i < Shape<T, DH>::KT * C / NT; ++i) {
        const int idx = tid + i * NT, row = idx / C, ch = idx % C;
        u32x4 z = {0, 0, 0, 0};
        if (r0 + row < end) z = *reinterpret_cast<const u32x4*>(base + (long)(r0 + row) * ld + ch * (16 / (int)sizeof(T)));
        *reinterpret_cast<u32x4*>(tile + row * ROW + ch * 16) = z;
    }
}
// acc[d][column] of this lane's column, times `mul`, to a row of DH elements.
template <typename T, int DH> __device__ __forceinline__ void put(T* row, const f32x16* acc, float mul, int lane) {
#pragma unroll
    for (int d = 0; d < DH / 32; ++d)
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            float x[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = acc[d][4 * b + e] * mul;
            Vec4<T>::store(row + 32 * d + 8 * b + 4 * (lane >> 5), x);
        }
}
// LDS written by other lanes of this wave may be read behind it (a wave's LDS accesses take effect in order).
__device__ __forceinline__ void wave_lds_fence() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}
__device__ __forceinline__ int length_of(const Slide& p, int b) {
    if (!p.lengths) return p.N;
    const int n = p.lengths[b];
    return n < 0 ? 0 : (n < p.N ? n : p.N);
}

// ----------------------------------------------------------------------------- softmax of a column, tile after tile
// m: running maximum of the raw scores, l: running sum of exp2((s - m) sc), this lane half's rows only until finish().
struct Softmax {
    float m = -INFINITY, l = 0.f;
    // s -> probabilities relative to the new maximum; returns the factor of everything before.
    __device__ __forceinline__ float step(f32x16& s, float sc) {
        float t = s[0];
#pragma unroll
        for (int r = 1; r < 16; ++r) t = fmaxf(t, s[r]);
        t = fmaxf(t, __shfl_xor(t, 32, 64));
        const float mn = fmaxf(m, t);
        const float nb = mn == -INFINITY ? 0.f : -mn * sc;         // nothing visible yet: every term is exp2(-inf) = 0
        const float alpha = __builtin_amdgcn_exp2f(__builtin_fmaf(m, sc, nb));
        float sum = 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            s[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], sc, nb));
            sum += s[r];
        }
        l = l * alpha + sum;
        m = mn;
        return alpha;
    }
    __device__ __forceinline__ float total() const { return l + __shfl_xor(l, 32, 64); }
};

// ----------------------------------------------------------------------------- forward
// One workgroup: 128 queries of one (sequence, head), each wave 32 of them; key tiles stream through LDS.
template <typename T, int DH, bool CAUSAL>
__global__ __launch_bounds__(256, 1) void slide_fwd_kernel(Slide p) {
    using S = Shape<T, DH>;
    extern __shared__ __align__(16) char lds[];
    char* Ks = lds;
    char* Vs = lds + S::KT * S::ROW;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int h = blockIdx.y, b = blockIdx.z, hk = h / p.G;
    const int n = length_of(p, b);
    const int q0 = blockIdx.x * TQ, qa = q0 + wave * 32, qi = qa + (lane & 31);
    const T* K = (const T*)p.k + b * p.k_b + hk * p.k_h;
    const T* V = (const T*)p.v + b * p.v_b + hk * p.v_h;
    Kept<T, DH> q;
    q.load((const T*)p.q + b * p.q_b + h * p.q_h + (long)qi * p.q_n, lane >> 5, qi < n);
    const float sc = p.scale * LOG2E;
    f32x16 acc[DH / 32] = {};
    Softmax sm;
    const Tiles tl = key_tiles<CAUSAL>(q0, q0 + TQ - 1, n, p.window, p.sinks, S::KT);
    for (int t = 0; t < tl.count(); ++t) {
        const int k0 = tl.at(t) * S::KT;
        __syncthreads();
        stage<T, DH, 256>(Ks, K, p.k_n, k0, n, tid);
        stage<T, DH, 256>(Vs, V, p.v_n, k0, n, tid);
        __syncthreads();
#pragma unroll
        for (int sub = 0; sub < S::KT; sub += 32) {
            const int ka = k0 + sub;
            const int cov = coverage<CAUSAL>(qa, qa + 31, ka, ka + 31, n, p.window, p.sinks);
            if (cov == 0) continue;
            f32x16 s = product<DH>(Ks, sub, q, lane);
            if (cov == 1) {
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (!visible<CAUSAL>(qi, ka + 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3), n, p.window, p.sinks)) s[r] = -INFINITY;
            }
            const float alpha = sm.step(s, sc);
#pragma unroll
            for (int d = 0; d < DH / 32; ++d) acc[d] *= alpha;
            gather<DH>(acc, Vs, sub, s, lane, T{});
        }
    }
    const float l = sm.total();
    if (qi < p.N) {
        const float inv = l > 0.f ? 1.f / l : 0.f;
        const long row = ((long)b * p.N + qi) * p.Hq + h;
        put<T, DH>((T*)p.o + row * DH, acc, inv, lane);
        if (p.o32) put<float, DH>(p.o32 + row * DH, acc, inv, lane);
        // base-2 logarithm of the row's sum; +inf for a row that sees nothing, so that backward's probabilities are 0
        if (p.lse && lane < 32) p.lse[((long)b * p.Hq + h) * p.N + qi] = l > 0.f ? sm.m * sc + __log2f(l) : INFINITY;
    }
}

// ----------------------------------------------------------------------------- backward
// delta = dO . o, one wave per four rows of a (sequence, head); o in 32 bits, so that what the rounded output lost is
// not multiplied by the cancellation in dP - delta.
template <typename T, int DH> __global__ __launch_bounds__(256) void slide_delta_kernel(Slide p, const float* o32) {
    const int lane = threadIdx.x & 15;
    const long r = (long)blockIdx.x * 16 + (threadIdx.x >> 4);           // (b, i, h)
    const long rows = (long)p.B * p.N * p.Hq;
    float s = 0.f;
    const int h = (int)(r % p.Hq);
    const long bi = r / p.Hq;
    const int i = (int)(bi % p.N), b = (int)(bi / p.N);
    if (r < rows && i < length_of(p, b)) {
        const T* d_o = (const T*)p.d_o + b * p.do_b + (long)i * p.do_n + h * p.do_h;
        const float* o = o32 + r * DH;
        for (int c = lane * 4; c < DH; c += 64) {
            float x[4], y[4];
            Vec4<T>::load(d_o + c, x);
            Vec4<float>::load(o + c, y);
            s += x[0] * y[0] + x[1] * y[1] + x[2] * y[2] + x[3] * y[3];
        }
    }
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    if (r < rows && lane == 0) p.delta[((long)b * p.Hq + h) * p.N + i] = s;
}

template <typename T, int DH, bool CAUSAL>
__global__ __launch_bounds__(256, 1) void slide_dq_kernel(Slide p) {
    using S = Shape<T, DH>;
    extern __shared__ __align__(16) char lds[];
    char* Ks = lds;
    char* Vs = lds + S::KT * S::ROW;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int h = blockIdx.y, b = blockIdx.z, hk = h / p.G;
    const int n = length_of(p, b);
    const int q0 = blockIdx.x * TQ, qa = q0 + wave * 32, qi = qa + (lane & 31);
    const T* K = (const T*)p.k + b * p.k_b + hk * p.k_h;
    const T* V = (const T*)p.v + b * p.v_b + hk * p.v_h;
    Kept<T, DH> q, d_o;
    q.load((const T*)p.q + b * p.q_b + h * p.q_h + (long)qi * p.q_n, lane >> 5, qi < n);
    d_o.load((const T*)p.d_o + b * p.do_b + h * p.do_h + (long)qi * p.do_n, lane >> 5, qi < n);
    const long st = ((long)b * p.Hq + h) * p.N + qi;
    const float lse = qi < n ? p.lse[st] : INFINITY, delta = qi < n ? p.delta[st] : 0.f;
    const float sc = p.scale * LOG2E;
    f32x16 acc[DH / 32] = {};
    const Tiles tl = key_tiles<CAUSAL>(q0, q0 + TQ - 1, n, p.window, p.sinks, S::KT);
    for (int t = 0; t < tl.count(); ++t) {
        const int k0 = tl.at(t) * S::KT;
        __syncthreads();
        stage<T, DH, 256>(Ks, K, p.k_n, k0, n, tid);
        stage<T, DH, 256>(Vs, V, p.v_n, k0, n, tid);
        __syncthreads();
#pragma unroll
        for (int sub = 0; sub < S::KT; sub += 32) {
            const int ka = k0 + sub;
            const int cov = coverage<CAUSAL>(qa, qa + 31, ka, ka + 31, n, p.window, p.sinks);
            if (cov == 0) continue;
            f32x16 s = product<DH>(Ks, sub, q, lane);
            const f32x16 dp = product<DH>(Vs, sub, d_o, lane);
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], sc, -lse)) * (dp[r] - delta);
                if (cov == 1 && !visible<CAUSAL>(qi, ka + 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3), n, p.window, p.sinks)) x = 0.f;
                s[r] = x;
            }
            gather<DH>(acc, Ks, sub, s, lane, T{});
        }
    }
    if (qi < p.N) put<T, DH>((T*)p.dq + b * p.dq_b + (long)qi * p.dq_n + h * p.dq_h, acc, qi < n ? p.scale : 0.f, lane);
}

// One workgroup: 128 keys of one (sequence, key head); the queries of every head that shares it stream through LDS.
template <typename T, int DH, bool CAUSAL>
__global__ __launch_bounds__(256, 1) void slide_dkv_kernel(Slide p) {
    using S = Shape<T, DH>;
    extern __shared__ __align__(16) char lds[];
    char* Qs = lds;
    char* Os = lds + S::KT * S::ROW;
    float* Ls = reinterpret_cast<float*>(lds + 2 * S::KT * S::ROW);     // [KT] lse, [KT] delta
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int hk = blockIdx.y, b = blockIdx.z;
    const int n = length_of(p, b);
    const int k0 = blockIdx.x * TQ, ka = k0 + wave * 32, kj = ka + (lane & 31);
    Kept<T, DH> k, v;
    k.load((const T*)p.k + b * p.k_b + hk * p.k_h + (long)kj * p.k_n, lane >> 5, kj < n);
    v.load((const T*)p.v + b * p.v_b + hk * p.v_h + (long)kj * p.v_n, lane >> 5, kj < n);
    const float sc = p.scale * LOG2E;
    f32x16 dk[DH / 32] = {}, dv[DH / 32] = {};
    const Tiles tl = query_tiles<CAUSAL>(k0, k0 + TQ - 1, n, p.window, p.sinks, S::KT);
    for (int g = 0; g < p.G; ++g) {
        const int h = hk * p.G + g;
        const T* Q = (const T*)p.q + b * p.q_b + h * p.q_h;
        const T* DO = (const T*)p.d_o + b * p.do_b + h * p.do_h;
        const long st = ((long)b * p.Hq + h) * p.N;
        for (int t = 0; t < tl.count(); ++t) {
            const int q0 = tl.at(t) * S::KT;
            __syncthreads();
            stage<T, DH, 256>(Qs, Q, p.q_n, q0, n, tid);
            stage<T, DH, 256>(Os, DO, p.do_n, q0, n, tid);
            if (tid < S::KT) {
                const int i = q0 + tid;
                Ls[tid] = i < n ? p.lse[st + i] : INFINITY;
                Ls[S::KT + tid] = i < n ? p.delta[st + i] : 0.f;
            }
            __syncthreads();
#pragma unroll
            for (int sub = 0; sub < S::KT; sub += 32) {
                const int qa = q0 + sub;
                const int cov = coverage<CAUSAL>(qa, qa + 31, ka, ka + 31, n, p.window, p.sinks);
                if (cov == 0) continue;
                f32x16 s = product<DH>(Qs, sub, k, lane);
                f32x16 dp = product<DH>(Os, sub, v, lane);
#pragma unroll
                for (int bb = 0; bb < 4; ++bb) {
                    const int r0 = sub + 8 * bb + 4 * (lane >> 5);
                    const f32x4 ls = *reinterpret_cast<const f32x4*>(Ls + r0);
                    const f32x4 de = *reinterpret_cast<const f32x4*>(Ls + S::KT + r0);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int r = 4 * bb + e;
                        float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], sc, -ls[e]));
                        if (cov == 1 && !visible<CAUSAL>(q0 + r0 + e, kj, n, p.window, p.sinks)) x = 0.f;
                        s[r] = x;
                        dp[r] = x * (dp[r] - de[e]);
                    }
                }
                gather<DH>(dv, Os, sub, s, lane, T{});
                gather<DH>(dk, Qs, sub, dp, lane, T{});
            }
        }
    }
    if (kj < p.N) {
        put<T, DH>((T*)p.dk + b * p.dk_b + (long)kj * p.dk_n + hk * p.dk_h, dk, kj < n ? p.scale : 0.f, lane);
        put<T, DH>((T*)p.dv + b * p.dv_b + (long)kj * p.dv_n + hk * p.dv_h, dv, kj < n ? 1.f : 0.f, lane);
    }
}

// ----------------------------------------------------------------------------- one token over a cache
struct Decode {
    const void* q; const void* k; const void* v; void* o; const int* lengths; float* ws;
    int B, cap, Hq, Hkv, G, splits;
    long q_b, q_h, k_b, k_n, k_h, v_b, v_n, v_h;
    int window, sinks;
    float scale;
};
// The heads that share a key head are the 32 MFMA columns.  Each wave stages its own 32 keys at a time (no barrier in
// the loop) and keeps a softmax of its own; the four are joined through LDS, the splits through the workspace:
// [B, Hq, splits] records of DH sums, a maximum (scaled, base 2) and a sum.
template <typename T, int DH>
__global__ __launch_bounds__(256, 1) void slide_decode_kernel(Decode p) {
    using S = Shape<T, DH>;
    extern __shared__ __align__(16) char lds[];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int groups = (p.G + 31) / 32;
    const int split = blockIdx.x, hk = blockIdx.y / groups, g0 = (blockIdx.y % groups) * 32, b = blockIdx.z;
    const int g = g0 + (lane & 31);
    int n = p.lengths[b];
    n = n < 0 ? 0 : (n < p.cap ? n : p.cap);
    char* Ks = lds + wave * 2 * 32 * S::ROW;
    char* Vs = Ks + 32 * S::ROW;
    const T* K = (const T*)p.k + b * p.k_b + hk * p.k_h;
    const T* V = (const T*)p.v + b * p.v_b + hk * p.v_h;
    Kept<T, DH> q;
    q.load((const T*)p.q + b * p.q_b + (long)(hk * p.G + g) * p.q_h, lane >> 5, g < p.G);
    const float sc = p.scale * LOG2E;
    f32x16 acc[DH / 32] = {};
    Softmax sm;
    const int back = n - p.window > 0 ? n - p.window : 0;              // first key of the window
    const int f = p.sinks < back ? p.sinks : back;                     // first tokens in front of it
    const int tf = (f + 31) / 32, tw = (n - back + 31) / 32;
    for (int t = split * 4 + wave; t < tf + tw; t += p.splits * 4) {
        const int k0 = t < tf ? t * 32 : back + (t - tf) * 32;
        const int end = t < tf ? f : n;
#pragma unroll
        for (int i = 0; i < 32 * S::CHUNKS / 64; ++i) {
            const int idx = lane + i * 64, row = idx / S::CHUNKS, ch = idx % S::CHUNKS;
            u32x4 x = {0, 0, 0, 0}, y = {0, 0, 0, 0};
            if (k0 + row < end) {
                x = *reinterpret_cast<const u32x4*>(K + (long)(k0 + row) * p.k_n + ch * (16 / (int)sizeof(T)));
                y = *reinterpret_cast<const u32x4*>(V + (long)(k0 + row) * p.v_n + ch * (16 / (int)sizeof(T)));
            }
            *reinterpret_cast<u32x4*>(Ks + row * S::ROW + ch * 16) = x;
            *reinterpret_cast<u32x4*>(Vs + row * S::ROW + ch * 16) = y;
        }
        wave_lds_fence();
        f32x16 s = product<DH>(Ks, 0, q, lane);
        if (k0 + 32 > end) {
#pragma unroll
            for (int r = 0; r < 16; ++r)
                if (k0 + 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3) >= end) s[r] = -INFINITY;
        }
        const float alpha = sm.step(s, sc);
#pragma unroll
        for (int d = 0; d < DH / 32; ++d) acc[d] *= alpha;
        gather<DH>(acc, Vs, 0, s, lane, T{});
        wave_lds_fence();
    }
    // the four waves' sums side by side: [wave][32 heads][DH + 2]
    float l = sm.total();
    const float m = sm.m == -INFINITY ? -INFINITY : sm.m * sc;
    __syncthreads();
    constexpr int W = DH + 4;
    float* out = reinterpret_cast<float*>(lds);
    float* mine = out + (wave * 32 + (lane & 31)) * W;
    put<float, DH>(mine, acc, 1.f, lane);
    if (lane < 32) { mine[DH] = m; mine[DH + 1] = l; }
    __syncthreads();
    for (int idx = tid; idx < 32 * DH; idx += 256) {
        const int c = idx / DH, d = idx % DH;
        if (g0 + c >= p.G) continue;
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < 4; ++w) top = fmaxf(top, out[(w * 32 + c) * W + DH]);
        float x = 0.f, sum = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float* rec = out + (w * 32 + c) * W;
            const float e = rec[DH] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(rec[DH] - top);
            x += rec[d] * e;
            sum += rec[DH + 1] * e;
        }
        const long row = (long)b * p.Hq + hk * p.G + g0 + c;
        if (p.splits == 1) {
            ((T*)p.o)[row * DH + d] = (T)(sum > 0.f ? x / sum : 0.f);
        } else {
            float* rec = p.ws + (row * p.splits + split) * (DH + 2);
            rec[d] = x;
            if (d == 0) { rec[DH] = top; rec[DH + 1] = sum; }
        }
    }
}
template <typename T, int DH> __global__ __launch_bounds__(DH < 64 ? 64 : DH) void slide_join_kernel(Decode p) {
    const long row = blockIdx.x;
    const int d = threadIdx.x;
    if (d >= DH) return;
    const float* rec = p.ws + row * p.splits * (DH + 2);
    float top = -INFINITY;
    for (int s = 0; s < p.splits; ++s) top = fmaxf(top, rec[s * (DH + 2) + DH]);
    float x = 0.f, sum = 0.f;
    for (int s = 0; s < p.splits; ++s) {
        const float* r = rec + s * (DH + 2);
        const float e = r[DH] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(r[DH] - top);
        x += r[d] * e;
        sum += r[DH + 1] * e;
    }
    ((T*)p.o)[row * DH + d] = (T)(sum > 0.f ? x / sum : 0.f);
}

// ----------------------------------------------------------------------------- host side
template <typename K> int allow_lds(K kernel, int bytes) {
    if (bytes <= 64 * 1024) return 0;
    return (int)hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
}
template <typename T, int DH, bool CAUSAL> int run_fwd(const Slide& p, hipStream_t st) {
    const int bytes = 2 * Shape<T, DH>::KT * Shape<T, DH>::ROW;
    if (int e = allow_lds(slide_fwd_kernel<T, DH, CAUSAL>, bytes)) return e;
    hipLaunchKernelGGL((slide_fwd_kernel<T, DH, CAUSAL>), dim3(vitk_ceil_div(p.N, TQ), p.Hq, p.B), dim3(256), bytes, st, p);
    VITK_CHECK_LAUNCH();
    return 0;
}
template <typename T, int DH, bool CAUSAL> int run_bwd(const Slide& p, const float* o32, hipStream_t st) {
    const int bytes = 2 * Shape<T, DH>::KT * Shape<T, DH>::ROW + 2 * Shape<T, DH>::KT * (int)sizeof(float);
    if (int e = allow_lds(slide_dq_kernel<T, DH, CAUSAL>, bytes)) return e;
    if (int e = allow_lds(slide_dkv_kernel<T, DH, CAUSAL>, bytes)) return e;
    const long rows = (long)p.B * p.N * p.Hq;
    hipLaunchKernelGGL((slide_delta_kernel<T, DH>), dim3((unsigned)((rows + 15) / 16)), dim3(256), 0, st, p, o32);
    VITK_CHECK_LAUNCH();
    const int tiles = vitk_ceil_div(p.N, TQ);
    if (p.dk) {
        hipLaunchKernelGGL((slide_dkv_kernel<T, DH, CAUSAL>), dim3(tiles, p.Hkv, p.B), dim3(256), bytes, st, p);
        VITK_CHECK_LAUNCH();
    }
    if (p.dq) {
        hipLaunchKernelGGL((slide_dq_kernel<T, DH, CAUSAL>), dim3(tiles, p.Hq, p.B), dim3(256), bytes, st, p);
        VITK_CHECK_LAUNCH();
    }
    return 0;
}
template <typename T, int DH> int run_decode(const Decode& p, hipStream_t st) {
    const int tiles = 4 * 2 * 32 * Shape<T, DH>::ROW, join = 4 * 32 * (DH + 4) * (int)sizeof(float);
    const int bytes = tiles > join ? tiles : join;
    if (int e = allow_lds(slide_decode_kernel<T, DH>, bytes)) return e;
    hipLaunchKernelGGL((slide_decode_kernel<T, DH>), dim3(p.splits, p.Hkv * ((p.G + 31) / 32), p.B), dim3(256), bytes, st, p);
    VITK_CHECK_LAUNCH();
    if (p.splits > 1) {
        hipLaunchKernelGGL((slide_join_kernel<T, DH>), dim3((unsigned)((long)p.B * p.Hq)), dim3(DH < 64 ? 64 : DH), 0, st, p);
        VITK_CHECK_LAUNCH();
    }
    return 0;
}

// 16-byte rows: the pointer and every stride.
bool aligned(const void* ptr, int esz, std::initializer_list<long> strides) {
    if ((uintptr_t)ptr % 16) return false;
    for (long s : strides)
        if (s * esz % 16) return false;
    return true;
}

int fill(const vitk_slide_attn* a, int dtype, bool backward, Slide& p) {
    if (!a || !a->q || !a->k || !a->v) return VITK_ERR_NULL;
    if (dtype != VITK_BF16 && dtype != VITK_F32) return VITK_ERR_DTYPE;
    if (a->dh != 32 && a->dh != 64 && a->dh != 128) return VITK_ERR_UNSUPPORTED;
    if (a->B <= 0 || a->N <= 0 || a->Hq <= 0 || a->Hkv <= 0 || a->Hq % a->Hkv || a->B > 65535 || a->Hq > 65535) return VITK_ERR_SHAPE;
    if (a->N > (1 << 30) || a->window < 0 || a->sinks < 0 || !(a->scale > 0.f)) return VITK_ERR_SHAPE;
    const int e = dtype == VITK_BF16 ? 2 : 4;
    if (!aligned(a->q, e, {a->q_b, a->q_n, a->q_h}) || !aligned(a->k, e, {a->k_b, a->k_n, a->k_h}) ||
        !aligned(a->v, e, {a->v_b, a->v_n, a->v_h})) return VITK_ERR_SHAPE;
    p = Slide{};
    p.q = a->q; p.k = a->k; p.v = a->v; p.o = a->o; p.o32 = a->o_f32; p.lse = a->lse; p.lengths = a->lengths;
    p.B = a->B; p.N = a->N; p.Hq = a->Hq; p.Hkv = a->Hkv; p.G = a->Hq / a->Hkv;
    p.q_b = a->q_b; p.q_n = a->q_n; p.q_h = a->q_h;
    p.k_b = a->k_b; p.k_n = a->k_n; p.k_h = a->k_h;
    p.v_b = a->v_b; p.v_n = a->v_n; p.v_h = a->v_h;
    p.window = a->window < a->N ? a->window : a->N;
    p.sinks = a->sinks < a->N ? a->sinks : a->N;
    p.scale = a->scale;
    if (!backward) {
        if (!a->o) return VITK_ERR_NULL;
        return aligned(a->o, e, {}) && aligned(a->o_f32, 4, {}) ? 0 : VITK_ERR_SHAPE;
    }
    if (!a->d_o || !a->lse || !a->delta || !a->dk != !a->dv || !(a->dq || a->dk)) return VITK_ERR_NULL;
    if (dtype == VITK_BF16 ? !a->o_f32 : !a->o) return VITK_ERR_NULL;
    if (!aligned(a->d_o, e, {a->do_b, a->do_n, a->do_h}) || !aligned(a->dq, e, {a->dq_b, a->dq_n, a->dq_h}) ||
        !aligned(a->dk, e, {a->dk_b, a->dk_n, a->dk_h}) || !aligned(a->dv, e, {a->dv_b, a->dv_n, a->dv_h})) return VITK_ERR_SHAPE;
    p.d_o = a->d_o; p.delta = a->delta; p.dq = a->dq; p.dk = a->dk; p.dv = a->dv;
    p.do_b = a->do_b; p.do_n = a->do_n; p.do_h = a->do_h;
    p.dq_b = a->dq_b; p.dq_n = a->dq_n; p.dq_h = a->dq_h;
    p.dk_b = a->dk_b; p.dk_n = a->dk_n; p.dk_h = a->dk_h;
    p.dv_b = a->dv_b; p.dv_n = a->dv_n; p.dv_h = a->dv_h;
    return 0;
}

}  // namespace

#define SLIDE_FORMS(CALL)                                                                                             \
    if (dtype == VITK_BF16) {                                                                                         \
        if (a->dh == 32) return a->causal ? CALL(bf16_t, 32, true) : CALL(bf16_t, 32, false);                         \
        if (a->dh == 64) return a->causal ? CALL(bf16_t, 64, true) : CALL(bf16_t, 64, false);                         \
        return a->causal ? CALL(bf16_t, 128, true) : CALL(bf16_t, 128, false);                                        \
    }                                                                                                                 \
    if (a->dh == 32) return a->causal ? CALL(float, 32, true) : CALL(float, 32, false);                               \
    if (a->dh == 64) return a->causal ? CALL(float, 64, true) : CALL(float, 64, false);                               \
    return a->causal ? CALL(float, 128, true) : CALL(float, 128, false)

extern "C" int vitk_slide_attn_fwd(const vitk_slide_attn* a, int dtype, void* stream) {
    Slide p;
    if (int e = fill(a, dtype, false, p)) return e;
    hipStream_t st = (hipStream_t)stream;
#define FWD(T, DH, C) run_fwd<T, DH, C>(p, st)
    SLIDE_FORMS(FWD);
}

extern "C" int vitk_slide_attn_bwd(const vitk_slide_attn* a, int dtype, void* stream) {
    Slide p;
    if (int e = fill(a, dtype, true, p)) return e;
    hipStream_t st = (hipStream_t)stream;
    const float* o32 = dtype == VITK_BF16 ? a->o_f32 : (const float*)a->o;
#define BWD(T, DH, C) run_bwd<T, DH, C>(p, o32, st)
    SLIDE_FORMS(BWD);
}

extern "C" int vitk_slide_decode(const vitk_slide_cache* a, int dtype, void* stream) {
    if (!a || !a->q || !a->k || !a->v || !a->o || !a->lengths) return VITK_ERR_NULL;
    if (dtype != VITK_BF16 && dtype != VITK_F32) return VITK_ERR_DTYPE;
    if (a->dh != 32 && a->dh != 64 && a->dh != 128) return VITK_ERR_UNSUPPORTED;
    if (a->B <= 0 || a->cap <= 0 || a->Hq <= 0 || a->Hkv <= 0 || a->Hq % a->Hkv || a->B > 65535) return VITK_ERR_SHAPE;
    if (a->cap > (1 << 30) || a->window < 0 || a->sinks < 0 || !(a->scale > 0.f) || a->splits < 1 || a->splits > 1024) return VITK_ERR_SHAPE;
    if (a->splits > 1 && !a->workspace) return VITK_ERR_NULL;
    const int e = dtype == VITK_BF16 ? 2 : 4;
    if (!aligned(a->q, e, {a->q_b, a->q_h}) || !aligned(a->k, e, {a->k_b, a->k_n, a->k_h}) || !aligned(a->v, e, {a->v_b, a->v_n, a->v_h}))
        return VITK_ERR_SHAPE;
    Decode p{};
    p.q = a->q; p.k = a->k; p.v = a->v; p.o = a->o; p.lengths = a->lengths; p.ws = a->workspace;
    p.B = a->B; p.cap = a->cap; p.Hq = a->Hq; p.Hkv = a->Hkv; p.G = a->Hq / a->Hkv; p.splits = a->splits;
    if ((long)p.Hkv * ((p.G + 31) / 32) > 65535) return VITK_ERR_SHAPE;
    p.q_b = a->q_b; p.q_h = a->q_h;
    p.k_b = a->k_b; p.k_n = a->k_n; p.k_h = a->k_h;
    p.v_b = a->v_b; p.v_n = a->v_n; p.v_h = a->v_h;
    p.window = a->window < a->cap ? a->window : a->cap;
    p.sinks = a->sinks < a->cap ? a->sinks : a->cap;
    p.scale = a->scale;
    hipStream_t st = (hipStream_t)stream;
    if (dtype == VITK_BF16) {
        if (a->dh == 32) return run_decode<bf16_t, 32>(p, st);
        if (a->dh == 64) return run_decode<bf16_t, 64>(p, st);
        return run_decode<bf16_t, 128>(p, st);
    }
    if (a->dh == 32) return run_decode<float, 32>(p, st);
    if (a->dh == 64) return run_decode<float, 64>(p, st);
    return run_decode<float, 128>(p, st);
}
