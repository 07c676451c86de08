// AdamW over a table of tensors: one pass for the gradients' norm, one for the update.
//
//   coef = min(1, max_norm / (|g| + 1e-6));  g' = coef g
//   m = b1 m + (1 - b1) g';  v = b2 v + (1 - b2) g'^2;  p = p (1 - lr wd) - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// HBM-bound: 4 bytes of every parameter for the norm, then 28 (states in 32 bits) or 16 + 16/256 (in 8), which leaves the
// 8-bit update about 90 vector instructions an element before it is bound by those instead.  A large copy reaches 5.0 TB/s;
// 87 million parameters in 32 bits: norm 99 us (3.5 TB/s), update 440 us (5.5 TB/s); 304 million in 8 bits: norm 236 us (5.2 TB/s),
// update 1005 us (4.8 TB/s), each launch by itself.
//
// States in 8 bits are e4m3 codes in units of a scale that 256 consecutive elements share (largest value / 448); the
// second moment is held as its root, which halves the range that the code has to span.  A code's neighbours are 1/16 to
// 1/8 of it apart and the second moment moves by a thousandth per step: rounded to nearest it would never move.  So
// codes are rounded at random, m in proportion to its distance from the two neighbours and v in proportion to the
// distance of their SQUARES (in proportion to the roots, E[v] would grow by the variance of the root at each step, more
// than the 1 - b2 that pulls it back).  A root that is not zero is never held as zero: the next step would divide by eps.
// What is no finite number (a gradient's NaN or infinity, a square beyond 32 bits) is held as the code's NaN, since there is none for
// infinity: it shows in its own parameter at the next step, and the other 255 elements keep their moments.
// The update itself uses the moments before they are rounded.  Nothing below is contracted, and
// sums have a fixed order, so codes, scales and parameters are the same bits wherever the same inputs are.
#include "common.h"

namespace {

#pragma clang fp contract(off)

constexpr int CHUNK = 8192;              // elements of a workgroup
constexpr int BLOCK = 256;               // elements that share a scale: one wave, four each
constexpr int PARTIALS = 8192;           // four turns of the workgroups that the chip holds: the last one is short
static_assert(1 + PARTIALS == VITK_ADAMW_SLOTS, "slots layout");
constexpr float TOP = 448.f;             // largest e4m3 value

struct Entry {                           // mirrors vitk_adamw_entry
    float* p; const float* g; void* m; void* v; float* ms; float* vs;
    long n;
    int block0;
    int flags;
};
static_assert(sizeof(Entry) == sizeof(vitk_adamw_entry), "table layout");

struct Consts { float b1, c1, b2, c2, decay, step, root, eps; uint32_t key; };

template <int WAVES> __device__ __forceinline__ double block_sum(double s) {
    __shared__ double part[WAVES];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
    __syncthreads();
    s = part[0];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) s += part[w];
    return s;
}

// A workgroup of any launch finds its tensor in `entry_of`: a search of the table is a chain of loads that a chunk of a
// small tensor does not outlast.
__global__ __launch_bounds__(256) void adamw_norm_kernel(const Entry* tab, const int* entry_of, int n_blocks, double* partial) {
    double s = 0.0;
    for (int blk = blockIdx.x; blk < n_blocks; blk += gridDim.x) {     // always in this order
        const Entry& en = tab[entry_of[blk]];
        const long base = (long)(blk - en.block0) * CHUNK;
        const int cnt = en.n - base < CHUNK ? (int)(en.n - base) : CHUNK;
        const float* g = en.g + base;
        const int whole = en.flags & 2 ? cnt & ~3 : 0;
        if (whole == CHUNK) {                                          // eight loads in flight
            f32x4 x[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) x[k] = *reinterpret_cast<const f32x4*>(g + threadIdx.x * 4 + k * 1024);
#pragma unroll
            for (int k = 0; k < 8; ++k)
                s += ((double)x[k][0] * x[k][0] + (double)x[k][1] * x[k][1]) + ((double)x[k][2] * x[k][2] + (double)x[k][3] * x[k][3]);
            continue;
        }
        for (int i = threadIdx.x * 4; i < whole; i += 1024) {
            const f32x4 x = *reinterpret_cast<const f32x4*>(g + i);
            s += ((double)x[0] * x[0] + (double)x[1] * x[1]) + ((double)x[2] * x[2] + (double)x[3] * x[3]);
        }
        for (int i = whole + threadIdx.x; i < cnt; i += 256) s += (double)g[i] * g[i];
    }
    s = block_sum<4>(s);
    if (threadIdx.x == 0) partial[blockIdx.x] = s;
}
// slots[0]: the factor of every gradient.  One workgroup, every partial sum in flight at once.
__global__ __launch_bounds__(1024) void adamw_norm_final_kernel(const double* partial, int nb, double max_norm, double* slots, float* norm) {
    constexpr int EACH = PARTIALS / 1024;
    double t[EACH] = {}, s = 0.0;
#pragma unroll
    for (int k = 0; k < EACH; ++k)
        if ((int)threadIdx.x + k * 1024 < nb) t[k] = partial[threadIdx.x + k * 1024];
#pragma unroll
    for (int k = 0; k < EACH; ++k) s += t[k];
    s = block_sum<16>(s);
    if (threadIdx.x == 0) {
        s = sqrt(s);
        const double r = max_norm / (s + 1e-6);
        slots[0] = r >= 1.0 ? 1.0 : r;                                 // a NaN stays one
        if (norm) *norm = (float)s;
    }
}

// FAST: the quotient of the update by a reciprocal of one unit's error, 2^-23 of an update that is itself a thousandth of the
// parameter; the full division's ten instructions an element show in the 8-bit step only.
template <bool FAST>
__device__ __forceinline__ void update(float& p, float g, float& m, float& v, float& root, float coef, const Consts& c) {
    g = g * coef;
    m = m * c.b1 + g * c.c1;
    v = v * c.b2 + (g * g) * c.c2;
    root = sqrtf(v);
    const float den = root * c.root + c.eps;
    p = p * c.decay - (FAST ? m * __builtin_amdgcn_rcpf(den) : m / den) * c.step;
}

__global__ __launch_bounds__(256) void adamw32_kernel(const Entry* tab, const int* entry_of, int first, const double* slots, Consts c) {
    const float coef = slots ? (float)slots[0] : 1.f;
    const int block = first + blockIdx.x;
    const Entry en = tab[entry_of[block]];
    const long base = (long)(block - en.block0) * CHUNK;
    const int cnt = en.n - base < CHUNK ? (int)(en.n - base) : CHUNK;
    float* p = en.p + base;
    const float* g = en.g + base;
    float* m = (float*)en.m + base;
    float* v = (float*)en.v + base;
    const bool fresh = en.flags & 1;
    const int whole = en.flags & 2 ? cnt & ~3 : 0;
    float root;
    for (int i = threadIdx.x * 4; i < whole; i += 1024) {
        f32x4 pv = *reinterpret_cast<const f32x4*>(p + i);
        const f32x4 gv = *reinterpret_cast<const f32x4*>(g + i);
        f32x4 mv = {0.f, 0.f, 0.f, 0.f}, vv = mv;
        if (!fresh) {
            mv = *reinterpret_cast<const f32x4*>(m + i);
            vv = *reinterpret_cast<const f32x4*>(v + i);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            float a = pv[k], b = mv[k], d = vv[k];
            update<false>(a, gv[k], b, d, root, coef, c);
            pv[k] = a; mv[k] = b; vv[k] = d;
        }
        *reinterpret_cast<f32x4*>(m + i) = mv;
        *reinterpret_cast<f32x4*>(v + i) = vv;
        *reinterpret_cast<f32x4*>(p + i) = pv;
    }
    for (int i = whole + threadIdx.x; i < cnt; i += 256) {
        float a = p[i], b = fresh ? 0.f : m[i], d = fresh ? 0.f : v[i];
        update<false>(a, g[i], b, d, root, coef, c);
        p[i] = a; m[i] = b; v[i] = d;
    }
}

// ----------------------------------------------------------------------------- 8-bit states
// The word of an element: 16 bits for the first moment, 16 for the second.
__device__ __forceinline__ uint32_t word_of(long e, uint32_t key) {
    return mix32((uint32_t)e ^ key ^ ((uint32_t)(e >> 32) * 0x9E3779B1U));
}
// (Values here are no NaNs: a comparison needs none of fminf()'s quieting.)
__device__ __forceinline__ float least(float a, float b) { return a < b ? a : b; }
// Codes of magnitude a <= 448 between 2^-6 and 448 have three bits behind the leading one; below 2^-6 they are
// multiples of 2^-9, which is what three bits are once 2^-6 is added.
__device__ __forceinline__ float code_m(float y, uint32_t r16) {
    float a = fabsf(y);
    const float less = a < 0.015625f ? 0.015625f : 0.f;
    const uint32_t b = (__float_as_uint(a + less) + (r16 << 4) + 8u) & ~0xFFFFFu;
    a = least(__uint_as_float(b) - less, TOP);
    return __uint_as_float(__float_as_uint(a) | (__float_as_uint(y) & 0x80000000u));
}
__device__ __forceinline__ float code_v(float y, uint32_t r16) {
    const float less = y < 0.015625f ? 0.015625f : 0.f;
    const uint32_t b = __float_as_uint(least(y, TOP) + less) & ~0xFFFFFu;
    const float lo = __uint_as_float(b) - less, hi = least(__uint_as_float(b + 0x100000u) - less, TOP);
    const float u = ((float)r16 + 0.5f) * 1.52587890625e-5f;
    const float l2 = lo * lo;
    const float a = u * (hi * hi - l2) < y * y - l2 ? hi : lo;
    return y > 0.f && a == 0.f ? 0.001953125f : a;
}
// The largest of a wave's non-negative values, by their bits (a NaN is larger than all), in registers.
template <int CTRL, int ROWS> __device__ __forceinline__ uint32_t larger(uint32_t x) {
    const uint32_t y = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 0xf, false);
    return x > y ? x : y;
}
__device__ __forceinline__ float wave_max(uint32_t x) {
    x = larger<0xB1, 0xf>(x);        // within four lanes: xor 1
    x = larger<0x4E, 0xf>(x);        // xor 2
    x = larger<0x124, 0xf>(x);       // within 16: rotated by 4
    x = larger<0x128, 0xf>(x);       // by 8
    x = larger<0x142, 0xa>(x);       // rows 1 and 3: the last lane of the row before
    x = larger<0x143, 0xc>(x);       // rows 2 and 3: lane 31
    return __uint_as_float(__builtin_amdgcn_readlane(x, 63));
}
template <bool VEC>
__device__ __forceinline__ void step8(const Entry& en, long base, int cnt, float coef, const Consts& c) {
    const int lane = threadIdx.x & 63;
    const bool fresh = en.flags & 1;
    for (int blk = threadIdx.x >> 6; blk * BLOCK < cnt; blk += 4) {
        const int i0 = blk * BLOCK + lane * 4;
        const long at = base + i0;
        const int left = cnt - i0;                       // this lane's elements: min(4, left)
        const bool whole = VEC && left >= 4;
        float p[4] = {}, g[4] = {}, m[4] = {}, v[4] = {}, root[4] = {};
        uint32_t mc = 0, vc = 0;
        if (whole) {
            Vec4<float>::load(en.p + at, p);
            Vec4<float>::load(en.g + at, g);
            if (!fresh) {
                mc = *reinterpret_cast<const uint32_t*>((const uint8_t*)en.m + at);
                vc = *reinterpret_cast<const uint32_t*>((const uint8_t*)en.v + at);
            }
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (k < left) {
                    p[k] = en.p[at + k];
                    g[k] = en.g[at + k];
                    if (!fresh) {
                        mc |= (uint32_t)((const uint8_t*)en.m)[at + k] << (8 * k);
                        vc |= (uint32_t)((const uint8_t*)en.v)[at + k] << (8 * k);
                    }
                }
        }
        const long sb = (base + blk * BLOCK) / BLOCK;
        const float ms = fresh ? 0.f : en.ms[sb], vs = fresh ? 0.f : en.vs[sb];
        m[0] = __builtin_amdgcn_cvt_f32_fp8(mc, 0); m[1] = __builtin_amdgcn_cvt_f32_fp8(mc, 1);
        m[2] = __builtin_amdgcn_cvt_f32_fp8(mc, 2); m[3] = __builtin_amdgcn_cvt_f32_fp8(mc, 3);
        v[0] = __builtin_amdgcn_cvt_f32_fp8(vc, 0); v[1] = __builtin_amdgcn_cvt_f32_fp8(vc, 1);
        v[2] = __builtin_amdgcn_cvt_f32_fp8(vc, 2); v[3] = __builtin_amdgcn_cvt_f32_fp8(vc, 3);
        uint32_t um = 0, uv = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            m[k] = m[k] * ms;
            v[k] = v[k] * vs;
            v[k] = v[k] * v[k];
            update<true>(p[k], g[k], m[k], v[k], root[k], coef, c);
            const uint32_t a = __float_as_uint(m[k]) & 0x7FFFFFFFu, b = __float_as_uint(root[k]);
            um = um > a ? um : a;
            uv = uv > b ? uv : b;
        }
        float tm = wave_max(um), tv = wave_max(uv);
        uint32_t mn = 0, vn = 0;                         // codes of NaN where a moment is no finite number
        if (!(tm < INFINITY && tv < INFINITY)) {         // the scales come from the others, which keep what they hold
            um = uv = 0;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint32_t a = __float_as_uint(m[k]) & 0x7FFFFFFFu, b = __float_as_uint(root[k]) & 0x7FFFFFFFu;
                if (a >= 0x7F800000u) { mn |= 0x7Fu << (8 * k); m[k] = 0.f; }
                else um = um > a ? um : a;
                if (b >= 0x7F800000u) { vn |= 0x7Fu << (8 * k); root[k] = 0.f; }
                else uv = uv > b ? uv : b;
            }
            tm = wave_max(um);
            tv = wave_max(uv);
        }
        const float im = tm >= 1.925929944387236e-34f ? TOP / tm : 0.f;          // 2^-112: nothing to hold
        const float iv = tv >= 1.925929944387236e-34f ? TOP / tv : 0.f;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const uint32_t w = word_of(at + k, c.key);
            m[k] = code_m(m[k] * im, w & 0xFFFFu);
            v[k] = code_v(root[k] * iv, w >> 16);
        }
        mc = __builtin_amdgcn_cvt_pk_fp8_f32(m[0], m[1], 0, false);
        mc = __builtin_amdgcn_cvt_pk_fp8_f32(m[2], m[3], mc, true);
        vc = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false);
        vc = __builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], vc, true);
        mc |= mn;
        vc |= vn;
        if (whole) {
            Vec4<float>::store(en.p + at, p);
            *reinterpret_cast<uint32_t*>((uint8_t*)en.m + at) = mc;
            *reinterpret_cast<uint32_t*>((uint8_t*)en.v + at) = vc;
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (k < left) {
                    en.p[at + k] = p[k];
                    ((uint8_t*)en.m)[at + k] = (uint8_t)(mc >> (8 * k));
                    ((uint8_t*)en.v)[at + k] = (uint8_t)(vc >> (8 * k));
                }
        }
        if (lane == 0) {
            en.ms[sb] = im > 0.f ? tm * (1.f / TOP) : 0.f;
            en.vs[sb] = iv > 0.f ? tv * (1.f / TOP) : 0.f;
        }
    }
}
__global__ __launch_bounds__(256) void adamw8_kernel(const Entry* tab, const int* entry_of, int first, const double* slots, Consts c) {
    const float coef = slots ? (float)slots[0] : 1.f;
    const int block = first + blockIdx.x;
    const Entry en = tab[entry_of[block]];
    const long base = (long)(block - en.block0) * CHUNK;
    const int cnt = en.n - base < CHUNK ? (int)(en.n - base) : CHUNK;
    if (en.flags & 2) step8<true>(en, base, cnt, coef, c);
    else step8<false>(en, base, cnt, coef, c);
}

uint32_t host_mix32(uint32_t x) {
    x ^= x >> 16; x *= 0x7feb352dU;
    x ^= x >> 15; x *= 0x846ca68bU;
    return x ^ (x >> 16);
}

}  // namespace

extern "C" int vitk_adamw_norm(const void* table, const int* entry_of, int n_blocks, double max_norm, double* slots, float* norm,
                               void* stream) {
    if (!table || !entry_of || !slots) return VITK_ERR_NULL;
    if (n_blocks <= 0 || !(max_norm >= 0.0)) return VITK_ERR_SHAPE;
    hipStream_t st = (hipStream_t)stream;
    const int nb = n_blocks < PARTIALS ? n_blocks : PARTIALS;
    hipLaunchKernelGGL(adamw_norm_kernel, dim3(nb), dim3(256), 0, st, (const Entry*)table, entry_of, n_blocks, slots + 1);
    VITK_CHECK_LAUNCH();
    hipLaunchKernelGGL(adamw_norm_final_kernel, dim3(1), dim3(1024), 0, st, slots + 1, nb, max_norm, slots, norm);
    VITK_CHECK_LAUNCH();
    return 0;
}

extern "C" int vitk_adamw_step(const void* table, const int* entry_of, int first_block, int n_blocks, const double* slots, double lr,
                               double beta1, double beta2, double eps, double weight_decay, long step, int state_bits,
                               uint32_t seed, void* stream) {
    if (!table || !entry_of) return VITK_ERR_NULL;
    if (first_block < 0 || n_blocks <= 0 || step < 1) return VITK_ERR_SHAPE;
    if (state_bits != 32 && state_bits != 8) return VITK_ERR_UNSUPPORTED;
    if (!(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0 && eps >= 0.0)) return VITK_ERR_SHAPE;
    Consts c{};
    c.b1 = (float)beta1; c.c1 = (float)(1.0 - beta1);
    c.b2 = (float)beta2; c.c2 = (float)(1.0 - beta2);
    c.decay = (float)(1.0 - lr * weight_decay);
    c.step = (float)(lr / (1.0 - pow(beta1, (double)step)));
    c.root = (float)(1.0 / sqrt(1.0 - pow(beta2, (double)step)));
    c.eps = (float)eps;
    c.key = host_mix32(seed + (uint32_t)step * 0x9E3779B1U);
    hipStream_t st = (hipStream_t)stream;
    if (state_bits == 32)
        hipLaunchKernelGGL(adamw32_kernel, dim3(n_blocks), dim3(256), 0, st, (const Entry*)table, entry_of, first_block, slots, c);
    else
        hipLaunchKernelGGL(adamw8_kernel, dim3(n_blocks), dim3(256), 0, st, (const Entry*)table, entry_of, first_block, slots, c);
    VITK_CHECK_LAUNCH();
    return 0;
}
