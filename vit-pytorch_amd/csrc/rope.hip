// Rotary positions with several axes: pair i of axis a turns by pos[a] * base^(-i / pairs[a]).
//
// Memory-bound: every element is read and written once, 3 operations each.  A workgroup takes a few tokens; the angles of
// a token are the same for all of its heads, so they are computed once, reduced to one turn in 64 bits (in 32 a position
// of a million has lost its fraction of a turn), and kept in LDS as cosines and sines while the heads stream past.
// 113 MB of bf16 read and as much written in 45 us, 206 MB of fp32 in 88 us (5.0 and 4.7 TB/s; a large copy reaches 4.9): 4 tokens a workgroup,
// which is 2 to 4 vectors a thread of heads like these.
#include "common.h"

namespace {

constexpr int MAX_PAIRS = 128;
constexpr int MAX_AXES = 8;

struct Rope {
    const void* x; void* y; const void* pos;
    long x_b, x_n, x_h, y_b, y_n, y_h, pos_b;
    int N, H, dh, P, axes, pos_kind;
    long tokens;                     // B * N
    long from;                       // the first of this launch
    float sign;
    int first[MAX_AXES + 1];         // pairs [first[a], first[a + 1]) belong to axis a
    double turns[MAX_PAIRS];         // turns per unit of position
};

__device__ __forceinline__ double position(const Rope& p, long at) {
    switch (p.pos_kind) {
        case 0: return (double)reinterpret_cast<const int64_t*>(p.pos)[at];
        case 1: return (double)reinterpret_cast<const int*>(p.pos)[at];
        case 2: return (double)reinterpret_cast<const float*>(p.pos)[at];
    }
    return reinterpret_cast<const double*>(p.pos)[at];
}

// V: elements moved at once, 16 bytes where pairs, strides and addresses allow it.  Half pairing: V pairs from two places V elements wide; interleaved: V / 2 pairs in a row.
template <typename T, int V, bool INTERLEAVED, int TOK>
__global__ __launch_bounds__(256) void rope_kernel(Rope p) {
    __shared__ float cs[TOK][MAX_PAIRS], sn[TOK][MAX_PAIRS];
    const long t0 = p.from + (long)blockIdx.x * TOK;
    const int toks = p.tokens - t0 < TOK ? (int)(p.tokens - t0) : TOK;
    for (int i = threadIdx.x; i < toks * p.P; i += 256) {
        const int t = i / p.P, pr = i - t * p.P;
        int a = 0;
        while (a + 1 < p.axes && pr >= p.first[a + 1]) ++a;
        const long tok = t0 + t, b = tok / p.N;
        double turn = position(p, b * p.pos_b + (tok - b * p.N) * p.axes + a) * p.turns[pr];
        turn -= rint(turn);
        float s, c;
        sincospif((float)(2.0 * turn), &s, &c);
        cs[t][pr] = c;
        sn[t][pr] = s * p.sign;
    }
    __syncthreads();
    const int rest = p.dh - 2 * p.P;
    const int turned = INTERLEAVED ? 2 * p.P / V : p.P / V, per = turned + rest / V;
    const int units = p.H * per;
    for (int u = threadIdx.x; u < toks * units; u += 256) {
        const int t = u / units, w = u - t * units, h = w / per, k = w - h * per;
        const long tok = t0 + t, b = tok / p.N, n = tok - b * p.N;
        const T* x = (const T*)p.x + b * p.x_b + n * p.x_n + h * p.x_h;
        T* y = (T*)p.y + b * p.y_b + n * p.y_n + h * p.y_h;
        typedef T vec __attribute__((ext_vector_type(V)));
        if (k >= turned) {
            const int d = 2 * p.P + (k - turned) * V;
            *reinterpret_cast<vec*>(y + d) = *reinterpret_cast<const vec*>(x + d);
        } else if constexpr (INTERLEAVED) {
            vec a = *reinterpret_cast<const vec*>(x + k * V);
#pragma unroll
            for (int i = 0; i < V; i += 2) {
                const float c = cs[t][(k * V + i) >> 1], s = sn[t][(k * V + i) >> 1];
                const float u0 = (float)a[i], u1 = (float)a[i + 1];
                a[i] = (T)(u0 * c - u1 * s);
                a[i + 1] = (T)(u1 * c + u0 * s);
            }
            *reinterpret_cast<vec*>(y + k * V) = a;
        } else {
            vec a = *reinterpret_cast<const vec*>(x + k * V), e = *reinterpret_cast<const vec*>(x + p.P + k * V);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float c = cs[t][k * V + i], s = sn[t][k * V + i];
                const float u0 = (float)a[i], u1 = (float)e[i];
                a[i] = (T)(u0 * c - u1 * s);
                e[i] = (T)(u1 * c + u0 * s);
            }
            *reinterpret_cast<vec*>(y + k * V) = a;
            *reinterpret_cast<vec*>(y + p.P + k * V) = e;
        }
    }
}

template <typename T, int V, bool I> int launch(Rope p, hipStream_t st) {
    constexpr int TOK = 4;
    constexpr long MOST = 1L << 23;          // workgroups of a launch, whose threads are counted in 32 bits
    for (; p.from < p.tokens; p.from += MOST * TOK) {
        const long blocks = (p.tokens - p.from + TOK - 1) / TOK;
        hipLaunchKernelGGL((rope_kernel<T, V, I, TOK>), dim3((unsigned)(blocks < MOST ? blocks : MOST)), dim3(256), 0, st, p);
        VITK_CHECK_LAUNCH();
    }
    return 0;
}
template <typename T, bool I> int by_width(const Rope& p, int v, hipStream_t st) {
    if constexpr (sizeof(T) == 2)
        if (v >= 8) return launch<T, 8, I>(p, st);
    if (v >= 4) return launch<T, 4, I>(p, st);
    if (v >= 2 || I) return launch<T, 2, I>(p, st);
    if constexpr (!I) return launch<T, 1, I>(p, st);
    return VITK_ERR_SHAPE;
}

}  // namespace

extern "C" int vitk_axial_rope(const vitk_rope* a, int dtype, void* stream) {
    if (!a || !a->x || !a->y || !a->pos) return VITK_ERR_NULL;
    if (dtype != VITK_BF16 && dtype != VITK_F32) return VITK_ERR_DTYPE;
    if (a->B <= 0 || a->N <= 0 || a->H <= 0 || a->dh <= 0 || a->dh > 2 * MAX_PAIRS || a->dh % 2) return VITK_ERR_SHAPE;
    if (a->axes < 1 || a->axes > MAX_AXES || a->pos_kind < 0 || a->pos_kind > 3 || !(a->base > 0.0)) return VITK_ERR_SHAPE;
    Rope p{};
    for (int k = 0; k < a->axes; ++k) {
        if (a->pairs[k] <= 0 || a->pairs[k] > a->dh / 2 - p.P) return VITK_ERR_SHAPE;
        for (int i = 0; i < a->pairs[k]; ++i)
            p.turns[p.P + i] = pow(a->base, -(double)i / a->pairs[k]) * 0.15915494309189533577;
        p.first[k] = p.P;
        p.P += a->pairs[k];
    }
    p.first[a->axes] = p.P;
    p.x = a->x; p.y = a->y; p.pos = a->pos;
    p.x_b = a->x_b; p.x_n = a->x_n; p.x_h = a->x_h;
    p.y_b = a->y_b; p.y_n = a->y_n; p.y_h = a->y_h;
    p.pos_b = a->pos_b;
    p.N = a->N; p.H = a->H; p.dh = a->dh; p.axes = a->axes; p.pos_kind = a->pos_kind;
    p.tokens = (long)a->B * a->N;
    if (p.tokens > (1L << 32)) return VITK_ERR_SHAPE;
    p.sign = a->inverse ? -1.f : 1.f;
    // the widest power of two that divides every place where a vector starts or ends
    const int e = dtype == VITK_BF16 ? 2 : 4;
    long all = a->x_b | a->x_n | a->x_h | a->y_b | a->y_n | a->y_h | (2 * p.P) | a->dh | (16 / e);
    if (!a->interleaved) all |= p.P;
    const uintptr_t ptrs = (uintptr_t)a->x | (uintptr_t)a->y;
    if (ptrs % e) return VITK_ERR_SHAPE;
    all |= (long)(ptrs / e);
    int v = (int)(all & -all);
    if (a->interleaved && v < 2) return VITK_ERR_SHAPE;
    hipStream_t st = (hipStream_t)stream;
    if (dtype == VITK_BF16) return a->interleaved ? by_width<bf16_t, true>(p, v, st) : by_width<bf16_t, false>(p, v, st);
    return a->interleaved ? by_width<float, true>(p, v, st) : by_width<float, false>(p, v, st);
}
