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
//
// Rows that see a window cost the same everywhere; the first tokens do not: every query looks at their keys, and without a
// causal mask they look at every key.  The workgroup of a tile therefore handles the tile's BAND only (its window and, for
// ordinary rows, the few first tokens on the other side), and what the first tokens see beyond their band is cut into
// chunks of FAR items: 32 first tokens against a share of the far rows, dealt out to four waves that meet in LDS.
// Bands and chunks of a first token leave 32-bit records in a workspace, which a last small launch adds in a fixed order; so do the
// workgroups that share a band of keys in the backward pass of few key heads.
// Where the whole sequence is not much longer than a band, one item does all of 32 first tokens and nothing is left to add.
// (Without the split the backward pass of 16384 causal tokens of the sizes below takes 659 us instead of 276.)
//
// Measured in bf16, training, replayed from graphs, rates of the pairs that are visible (4 dh operations each forward, 6 for dQ, 8 for
// dK / dV, whose time is what they add to a backward pass):
//   8 x 2305 x 12 x 64, all visible:            forward 184 us (711 TFLOP/s), dQ 228 (860), dK / dV 298 (877)
//   1 x 16384 x 8 of 2 x 128, causal, window 1024:     87 us (766),               112 (895),          164 (815)
//   8 x 2305 x 12 x 64, window 145, 1 first token:     52 us (310),                64 (372),           78 (407)
// In the last, whose band is little longer than its rows, 127 MB forward and 353 MB backward are half of the time at the rate of a
// copy.  Every such time below is of the same run: of whole launches back to back, replayed.
#include <initializer_list>

#include "common.h"

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr float LOG2E = 1.4426950408889634f;
constexpr int TQ = 128;                       // rows of a workgroup: four waves of 32

struct Slide {
    const void* q; const void* k; const void* v; void* o; int8_t* rest; float* lse; const int* lengths;
    const void* d_o; float* delta; void* dq; void* dk; void* dv;
    int B, N, Hq, Hkv, G;
    long q_b, q_n, q_h, k_b, k_n, k_h, v_b, v_n, v_h, do_b, do_n, do_h, dq_b, dq_n, dq_h, dk_b, dk_n, dk_h, dv_b, dv_n, dv_h;
    int window, sinks;
    float scale;
    int single;                // whether every query sees one key only, however long the sequence
    int rows;                  // first tokens in items of their own, a multiple of 32 (0: none)
    int chunks;                // far items of each 32 of them; a row has chunks + 1 records, the band's last.  0: one item
                               // for all that 32 of them see, and no records
    float* ws;                 // forward: records of dh + 2; backward: dk | dv, then dq, records of dh
    float* ws_q;
    float* ws_b;               // of dK / dV bands that `shares` workgroups have in common: records of dk | dv, one of each share
    int shares;
    int far_items, items;      // of this launch: far ones come first, then bands
};

// ----------------------------------------------------------------------------- which pairs are visible
// What one row sees of the other axis: len rows from lo on, and the rows before f.
struct Span {
    int lo, len, f;
    __device__ __forceinline__ bool sees(int x) const { return (unsigned)(x - lo) < (unsigned)len || x < f; }
};
__device__ __forceinline__ Span span(int lo, int hi, int f) { return Span{lo, hi >= lo ? hi - lo + 1 : 0, f}; }
__device__ __forceinline__ int least(int a, int b) { return a < b ? a : b; }
template <bool CAUSAL> __device__ __forceinline__ Span keys_of(int i, int n, int w, int f) {
    if (i >= n) return Span{0, 0, 0};
    if (CAUSAL) return span(w > 0 ? i - w + 1 : i + 1, i, least(f, i + 1));
    if (i < f) return Span{0, n, 0};
    return span(w > 0 ? i - w + 1 : n, least(i + w, n) - 1, least(f, n));
}
template <bool CAUSAL> __device__ __forceinline__ Span queries_of(int j, int n, int w, int f) {
    if (j >= n) return Span{0, 0, 0};
    if (CAUSAL) return span(j, j < f ? n - 1 : least(j + w, n) - 1, 0);
    if (j < f) return Span{0, n, 0};
    return span(w > 0 ? j - w + 1 : n, least(j + w, n) - 1, least(f, n));
}
// s[r] of the rows that are not seen; register r holds row x0 + 8 (r / 4) + r % 4.  `first`: whether rows before f may be
// among them.
__device__ __forceinline__ void hide(f32x16& s, const Span& v, int x0, bool first, float with) {
    asm volatile("");          // a branch, not selects: most tiles have nothing to hide
    const int d = x0 - v.lo;
    if (first) {
#pragma unroll
        for (int r = 0; r < 16; ++r)
            if (!v.sees(x0 + 8 * (r >> 2) + (r & 3))) s[r] = with;
    } else {
#pragma unroll
        for (int r = 0; r < 16; ++r)
            if ((unsigned)(d + 8 * (r >> 2) + (r & 3)) >= (unsigned)v.len) s[r] = with;
    }
}
// What 32 rows see of 32 rows [x, x + 31] of the other axis: 0 nothing, 2 everything, 1 some pairs.  Rows [lo, hi] are seen by
// some of them and rows [flo, fhi] by all; of the rows before f some are seen, those before ff by all.  Four comparisons of
// scalars a tile: what the general test of a rectangle costs showed in the time of the loops.
struct Cover {
    int lo, hi, flo, fhi, f, ff;
    __device__ __forceinline__ int of(int x) const {
        if (x >= f && (x + 31 < lo || x > hi)) return 0;
        return (x >= flo && x + 31 <= fhi) || x + 31 < ff ? 2 : 1;
    }
};
__device__ __forceinline__ Cover only_some(Cover c, bool some) {      // nothing is seen by all
    if (some) { c.flo = c.fhi + 1; c.ff = 0; }
    return c;
}
// Of keys, by queries [a, a + 31]; no key is seen by a query behind the sequence.
template <bool CAUSAL> __device__ __forceinline__ Cover keys_by(int a, int n, int w, int f) {
    if (a >= n) return Cover{n, -1, n, -1, 0, 0};
    const int z = a + 31, r = w > 0 ? w - 1 : -1;
    f = least(f, n);
    if (CAUSAL)
        return only_some(Cover{a - r, w > 0 ? least(z, n - 1) : -1, z - r, w > 0 ? least(a, n - 1) : -1, least(f, z + 1), least(f, a + 1)}, z >= n);
    if (a < f) return only_some(Cover{0, n - 1, z < f ? 0 : z - r, z < f ? n - 1 : least(a + r, n - 1), f, f}, z >= n);
    return only_some(Cover{a - r, least(z + r, n - 1), z - r, least(a + r, n - 1), f, f}, z >= n);
}
// Of queries, by keys [a, a + 31].
template <bool CAUSAL> __device__ __forceinline__ Cover queries_by(int a, int n, int w, int f) {
    if (a >= n) return Cover{n, -1, n, -1, 0, 0};
    const int z = a + 31, r = w > 0 ? w - 1 : -1;
    f = least(f, n);
    if (CAUSAL) return only_some(Cover{a, a < f ? n - 1 : least(z + r, n - 1), z, z < f ? n - 1 : least(a + r, n - 1), 0, 0}, z >= n);
    if (a < f) return only_some(Cover{0, n - 1, z < f ? 0 : z - r, z < f ? n - 1 : least(a + r, n - 1), f, f}, z >= n);
    return only_some(Cover{a - r, least(z + r, n - 1), z - r, least(a + r, n - 1), f, f}, z >= n);
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
// The band of query rows [qa, qb], of key rows [ka, kb].  A window of 0 is listed like one of 1, so that far rows always lie
// behind the diagonal.
template <bool CAUSAL> __device__ __forceinline__ Tiles key_tiles(int qa, int qb, int n, int w, int f, int T) {
    if (qa >= n) return Tiles{0, 0, 0};
    qb = qb < n ? qb : n - 1;
    const int r = (w > 1 ? w : 1) - 1;
    return tiles_of(qa - r, CAUSAL ? qb : qb + r, CAUSAL && f > qb + 1 ? qb + 1 : f, n, T);
}
template <bool CAUSAL> __device__ __forceinline__ Tiles query_tiles(int ka, int kb, int n, int w, int f, int T) {
    if (ka >= n) return Tiles{0, 0, 0};
    kb = kb < n ? kb : n - 1;
    const int r = (w > 1 ? w : 1) - 1;
    return tiles_of(CAUSAL ? ka : ka - r, kb + r, CAUSAL ? 0 : f, n, T);
}

// ----------------------------------------------------------------------------- operands
// An LDS tile: rows one behind the other, the 16-byte chunks of a row in an order of its own, so that what 16 lanes read
// side by side lies in all 64 banks: chunk c of row r at place c ^ mix(r).  Read are one chunk of 16 rows in a row (all
// mixes of 16 rows differ, as far as a row has chunks), and, transposed, 64 bytes of four rows (bf16: the mixes of rows
// 0 ... 3 differ in the bits above those 64 bytes) or 128 bytes of rows r and r + 4 (fp32).
template <typename T, int DH> struct Shape {
    static constexpr int ROW = DH * (int)sizeof(T);
    static constexpr int CHUNKS = ROW / 16;
    // Rows of a staged tile.  In fp32, 64 rows of a head of 32 (4 x 4099 causal tokens, 16 heads of 8, window 512, backward: 605 us, with 32 rows
    // 640), but 32 of a head of 64, whose tiles of 64 would leave two workgroups a CU (8 images of 2305 tokens: 977 us, with 64 rows 1017; the
    // causal tokens 1280 and 1222).
    static constexpr int KT = ROW <= 128 || sizeof(T) == 2 ? 64 : 32;
    static constexpr int PER = ROW >= 256 ? 1 : 256 / ROW;        // rows in 64 banks
    static __device__ __forceinline__ int mix(int r) {
        if constexpr (sizeof(T) == 2) return ((r & 3) / PER << 2) | ((r >> 2) & 3);
        else if constexpr (PER == 2) return (r >> 1) & 7;
        else return ((r >> 2) & 1) << 3 | ((r >> 3) & 1) << 2 | (r & 3);
    }
    static __device__ __forceinline__ int at(int r, int chunk) { return r * ROW + ((chunk ^ mix(r)) << 4); }
};
// x has arrived.  Without this the compiler would wait for it at its first use inside a loop, and with it, at every turn, for
// all that the loop has on its way into LDS.
template <typename X> __device__ __forceinline__ void arrived(X& x) { asm volatile("" : "+v"(x)); }
// The order of a run of N products that each read READS times from LDS: a few reads ahead of the products.
template <int N, int READS> __device__ __forceinline__ void reads_ahead() {
    constexpr int AHEAD = N < 4 ? N : 4;
    __builtin_amdgcn_sched_group_barrier(0x100, AHEAD * READS, 0);
#pragma unroll
    for (int i = 0; i < N - AHEAD; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, AHEAD, 0);
}
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
    __device__ __forceinline__ void settle() {
#pragma unroll
        for (int c = 0; c < DH / 16; ++c) arrived(f[c]);
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
    __device__ __forceinline__ void settle() {
#pragma unroll
        for (int i = 0; i < DH / 2; ++i) arrived(f[i]);
    }
};
// 32 tile rows from r0 times the kept rows, over the head, on top of acc: C[row][column].
template <int DH> __device__ __forceinline__ f32x16 product(const char* tile, int r0, const Kept<bf16_t, DH>& kept, int lane, f32x16 acc = {}) {
    const int a = Shape<bf16_t, DH>::at(lane & 31, lane >> 5);
    tile += r0 * Shape<bf16_t, DH>::ROW;
#pragma unroll
    for (int c = 0; c < DH / 16; ++c)
        acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(*reinterpret_cast<const bf16x8*>(tile + (a ^ (c << 5))), kept.f[c], acc, 0, 0, 0);
    reads_ahead<DH / 16, 1>();
    return acc;
}
// The same with the kept rows in an LDS tile.
template <typename T, int DH> struct KeptInLds { const char* rows; };
template <int DH> __device__ __forceinline__ f32x16 product(const char* tile, int r0, const KeptInLds<bf16_t, DH>& kept, int lane, f32x16 acc = {}) {
    const int a = Shape<bf16_t, DH>::at(lane & 31, lane >> 5);
    tile += r0 * Shape<bf16_t, DH>::ROW;
#pragma unroll
    for (int c = 0; c < DH / 16; ++c)
        acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(*reinterpret_cast<const bf16x8*>(tile + (a ^ (c << 5))),
                                                      *reinterpret_cast<const bf16x8*>(kept.rows + (a ^ (c << 5))), acc, 0, 0, 0);
    reads_ahead<DH / 16, 2>();
    return acc;
}
template <int DH> __device__ __forceinline__ f32x16 product(const char* tile, int r0, const Kept<float, DH>& kept, int lane, f32x16 acc = {}) {
    const int a = Shape<float, DH>::at(lane & 31, (lane >> 5) * (DH / 8));
    tile += r0 * Shape<float, DH>::ROW;
#pragma unroll
    for (int t = 0; t < DH / 8; ++t) {
        const f32x4 x = *reinterpret_cast<const f32x4*>(tile + (a ^ (t << 4)));
#pragma unroll
        for (int i = 0; i < 4; ++i) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(x[i], kept.f[4 * t + i], acc, 0, 0, 0);
    }
    return acc;
}
// acc[d][column] += sum over 32 tile rows from r0 of tile[row][d] * w[row][column]; w as a product left it.  In bf16
// the weights are rounded to the operand type here: by up to 2^-8 of each, independent, and the sums stay in 32 bits; FINE: what
// that leaves of them is a second operand.
template <int DH, bool FINE = false> __device__ __forceinline__ void gather(f32x16* acc, const char* tile, int r0, const f32x16& w, int lane, bf16_t) {
    using S = Shape<bf16_t, DH>;
    const int l15 = lane & 15, g = lane >> 4;
    bf16x8 b[2], rest[2];
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            b[c][e] = (bf16_t)w[8 * c + e];
            if constexpr (FINE) rest[c][e] = (bf16_t)(w[8 * c + e] - (float)b[c][e]);
        }
    // the transposing read takes 8 bytes of rows r ... r + 3 from each 16 lanes
    const int r = 4 * (g >> 1) + (l15 >> 2), ch = 2 * (g & 1) + ((l15 & 3) >> 1), half = (l15 & 1) * 8;
    const int a0 = S::at(r, ch) + half, a1 = S::at(r + 8, ch) + half;
    tile += r0 * S::ROW;
#pragma unroll
    for (int d = 0; d < DH / 32; ++d) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const char* t = tile + 16 * c * S::ROW;
            const bf16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((VITK_LDS bf16x4*)(t + (a0 ^ (d << 6))));
            const bf16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((VITK_LDS bf16x4*)(t + (a1 ^ (d << 6))));
            const bf16x8 a = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
            acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b[c], acc[d], 0, 0, 0);
            if constexpr (FINE) acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, rest[c], acc[d], 0, 0, 0);
        }
    }
    if constexpr (!FINE) reads_ahead<DH / 16, 2>();
}
template <int DH, bool FINE = false> __device__ __forceinline__ void gather(f32x16* acc, const char* tile, int r0, const f32x16& w, int lane, float) {
    using S = Shape<float, DH>;
    const int ch = (lane & 31) >> 2, low = (lane & 3) * 4;
    tile += r0 * S::ROW;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        const int a = S::at(8 * (r >> 2) + 4 * (lane >> 5) + (r & 3), ch) + low;
#pragma unroll
        for (int d = 0; d < DH / 32; ++d)
            acc[d] = __builtin_amdgcn_mfma_f32_32x32x2f32(*reinterpret_cast<const float*>(tile + (a ^ (d << 7))), w[r], acc[d], 0, 0, 0);
    }
}
// Rows behind the last one of the sequence are staged as that one again: finite, and without weight.
//
// Straight into LDS, 16 bytes a lane in the order of the lanes: each lane fetches the chunk that belongs at its place.  By all
// four waves (`voff`: where this thread's chunks lie from the tile's first row on.
// A base for them: moved by a scalar instruction, which waits for a vector instruction that may have made it, as the loads in
// assembly would not.
template <typename X> __device__ __forceinline__ const X* settled(const X* p) {
    const X* q;
    asm volatile("s_mov_b64 %0, %1" : "=s"(q) : "s"(p));
    return q;
}
__device__ __forceinline__ void dma16(const void* base, int off, unsigned lds) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(lds) : "memory");
}
__device__ __forceinline__ void dma4(const void* from, unsigned lds) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 4\n\tglobal_load_lds_dword %0, off" ::"v"(from), "s"(lds) : "memory");
}
__device__ __forceinline__ void dma_wait() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
__device__ __forceinline__ unsigned lds_addr(const void* p) { return (unsigned)(size_t)(VITK_LDS const char*)p; }
template <typename T, int DH, int NT = 256> struct Stage {
    using S = Shape<T, DH>;
    static constexpr int PARTS = S::KT * S::CHUNKS / NT;
    int voff[PARTS];
    int ld;
    __device__ __forceinline__ static int place(int i, int tid) { return i * NT + tid; }
    __device__ __forceinline__ int offset(int i, int tid, int last) const {
        const int pl = place(i, tid), r = pl / S::CHUNKS, ch = (pl % S::CHUNKS) ^ S::mix(r);
        return (r < last ? r : last) * ld * (int)sizeof(T) + ch * 16;
    }
    __device__ __forceinline__ Stage(long stride, int tid) : ld((int)stride) {
#pragma unroll
        for (int i = 0; i < PARTS; ++i) voff[i] = offset(i, tid, S::KT);
    }
    __device__ __forceinline__ void start(char* tile, const T* base, int r0, int n, int tid) const {
        const T* from = settled(base + (long)r0 * ld);
        const unsigned to = __builtin_amdgcn_readfirstlane(lds_addr(tile) + (tid & ~63) * 16);
        if (r0 + S::KT <= n) {
#pragma unroll
            for (int i = 0; i < PARTS; ++i) dma16(from, voff[i], to + i * NT * 16);
        } else {
#pragma unroll
            for (int i = 0; i < PARTS; ++i) dma16(from, offset(i, tid, n - 1 - r0), to + i * NT * 16);
        }
    }
};
// By one wave, through its registers.
template <typename T, int DH> struct Fetch {
    using S = Shape<T, DH>;
    u32x4 x[32 * S::CHUNKS / 64];
    __device__ __forceinline__ void load(const T* base, long ld, int r0, int n, int lane) {
#pragma unroll
        for (int i = 0; i < 32 * S::CHUNKS / 64; ++i) {
            const int idx = lane + i * 64, r = r0 + idx / S::CHUNKS;
            x[i] = *reinterpret_cast<const u32x4*>(base + (long)(r < n ? r : n - 1) * ld + idx % S::CHUNKS * (16 / (int)sizeof(T)));
        }
    }
    __device__ __forceinline__ void store(char* tile, int lane) const {
#pragma unroll
        for (int i = 0; i < 32 * S::CHUNKS / 64; ++i) {
            const int idx = lane + i * 64;
            *reinterpret_cast<u32x4*>(tile + S::at(idx / S::CHUNKS, idx % S::CHUNKS)) = x[i];
        }
    }
};
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
// LDS written by other lanes of this wave may be read behind it (a wave's LDS instructions take effect in order).
__device__ __forceinline__ void wave_lds_fence() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}
// The same towards copies that go straight into LDS: those write when memory answers, in no order with LDS instructions, so what
// this wave has read of the tile has to have arrived before the next one is asked for.
__device__ __forceinline__ void wave_reads_done() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }
// What rounding x to bf16 left, in units of 1/256 of the last place: with it an output has 15 bits behind the leading one, in
// 8 bits more of memory (o in 32 bits beside it would be 3 bytes an element more to write, keep and read).
__device__ __forceinline__ int rest_of(float x) {
    const int r = (int)(__float_as_uint(x) - ((unsigned)__builtin_bit_cast(unsigned short, (bf16_t)x) << 16));
    return least((r + 128) >> 8, 127);
}
// The wave's 32 rows, `ld` elements apart, the first `count` of them, through its LDS tile `via`: a lane's elements of a row are 4 here
// and 4 there, and rows written from registers cost the address units a line for each of them (8 images of 2305 tokens, window 145, backward: 143 us,
// from registers 150; 16384 tokens: no difference).
template <int DH> __device__ __forceinline__ void put_rows(char* via, bf16_t* rows, long ld, int count, const f32x16* acc, float mul, int lane) {
    using S = Shape<bf16_t, DH>;
#pragma unroll
    for (int d = 0; d < DH / 32; ++d)
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            bf16x4 x;
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = (bf16_t)(acc[d][4 * b + e] * mul);
            *reinterpret_cast<bf16x4*>(via + S::at(lane & 31, 4 * d + b) + 8 * (lane >> 5)) = x;
        }
    wave_lds_fence();
#pragma unroll
    for (int i = 0; i < 32 * S::CHUNKS / 64; ++i) {
        const int idx = lane + i * 64, r = idx / S::CHUNKS, c = idx % S::CHUNKS;
        if (r < count) *reinterpret_cast<u32x4*>(rows + r * ld + 8 * c) = *reinterpret_cast<const u32x4*>(via + S::at(r, c));
    }
    wave_lds_fence();
}
template <int DH> __device__ __forceinline__ void put_rows(char*, float* rows, long ld, int count, const f32x16* acc, float mul, int lane) {
    if ((lane & 31) < count) put<float, DH>(rows + (lane & 31) * ld, acc, mul, lane);
}
// The same of what their rounding left.
template <int DH> __device__ __forceinline__ void put_rest(char* via, int8_t* rows, long ld, int count, const f32x16* acc, float mul, int lane) {
    constexpr int CHUNKS = DH / 16;
    const auto at = [](int r, int c) { return r * DH + ((c ^ ((r >> 2) & (CHUNKS - 1))) << 4); };
#pragma unroll
    for (int d = 0; d < DH / 32; ++d)
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            unsigned x = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) x |= (unsigned)(rest_of(acc[d][4 * b + e] * mul) & 255) << (8 * e);
            *reinterpret_cast<unsigned*>(via + at(lane & 31, 2 * d + (b >> 1)) + 8 * (b & 1) + 4 * (lane >> 5)) = x;
        }
    wave_lds_fence();
#pragma unroll
    for (int i = 0; i < 32 * CHUNKS / 64; ++i) {
        const int idx = lane + i * 64, r = idx / CHUNKS, c = idx % CHUNKS;
        if (r < count) *reinterpret_cast<u32x4*>(rows + r * ld + 16 * c) = *reinterpret_cast<const u32x4*>(via + at(r, c));
    }
}
// What the sums of dQ and dK are multiplied with.  A query that sees one key only has the probability 1 whatever its score:
// where all do, the gradients of the scores are exactly 0, and not what dP - delta leaves after rounding.
__device__ __forceinline__ float score_scale(const Slide& p, int n) { return p.single || n == 1 ? 0.f : p.scale; }
__device__ __forceinline__ int length_of(const Slide& p, int b) {
    if (!p.lengths) return p.N;
    const int n = p.lengths[b];
    return n < 0 ? 0 : (n < p.N ? n : p.N);
}

// ----------------------------------------------------------------------------- softmax of a column, tile after tile
// m: a maximum of the raw scores, l: running sum of exp2((s - m) sc), of this lane half's rows only until total().
// fmaxf() would quiet every input first.  The compiler does not wait for a matrix instruction's result in front of assembly:
// `a` has to come from an instruction of its own that read the same result.
__device__ __forceinline__ float max3_raw(float a, float b, float c) {
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}
struct Softmax {
    float m = -INFINITY, l = 0.f;
    // Scores -> probabilities relative to m.  m follows the maximum only once that is 8 binary orders above it (in some
    // column of the wave): until then probabilities stay below 2^8, and the accumulators need no factor, which for a head
    // of 128 costs more than the exponentials.  `rescale(alpha)` applies it to everything before.
    template <typename F> __device__ __forceinline__ void step(f32x16& s, float sc, F rescale) {
        float t = fmaxf(s[0], s[1]);
#pragma unroll
        for (int r = 2; r < 16; r += 2) t = max3_raw(t, s[r], s[r + 1]);
        if (__any(t * sc > m * sc + 8.f)) {           // a row that has seen nothing: 0 > -inf, or -inf > -inf, which waits
            t = fmaxf(t, __shfl_xor(t, 32, 64));
            const float mn = fmaxf(m, t);
            const float alpha = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m - mn) * sc);
            l *= alpha;
            m = mn;
            rescale(alpha);
        }
        const float nb = m == -INFINITY ? 0.f : -m * sc;          // nothing visible yet: every term is exp2(-inf) = 0
        float sum = 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            s[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], sc, nb));
            sum += s[r];
        }
        l += sum;
    }
    __device__ __forceinline__ float total() const { return l + __shfl_xor(l, 32, 64); }
};

// ----------------------------------------------------------------------------- work items
// Far items first (the longest), then bands, a head's tiles in a row.  Workgroups go round the 8 XCDs in turn: each XCD
// gets a run of neighbouring items, whose tiles of the other axis it finds in its own L2.
struct Item { bool far, none; int x, h, b; };
__device__ __forceinline__ Item item_of(const Slide& p, int heads, int tiles) {
    Item it{};
    const int id = blockIdx.x;
    it.far = id < p.far_items;
    int k;
    if (it.far) {
        k = id;
        tiles = (p.chunks ? p.chunks : 1) * (p.rows / 32);
    } else {
        const int m = p.items - p.far_items, each = (m + 7) / 8, r = id - p.far_items;
        k = (r & 7) * each + (r >> 3);
        it.none = (r >> 3) >= each || k >= m;
    }
    it.x = k % tiles;
    it.h = k / tiles % heads;
    it.b = k / tiles / heads;
    return it;
}
// The factor of a record whose maximum is m, towards the common maximum.  Where both are -inf its sums are 0, or NaN if all
// that it looked at was: either way they stay what they are.  A record with a total of exactly 0 saw nothing: whatever its sums are (0
// times a NaN in v that another row of the item looked at), they do not count.
__device__ __forceinline__ float weight_of(float m, float top) { return m == top ? 1.f : __builtin_amdgcn_exp2f(m - top); }
__device__ __forceinline__ float counted(float x, float total, float weight) { return total == 0.f ? 0.f : x * weight; }
// A row's result from its sums; a total of exactly 0 is a row that sees nothing (a NaN is not).
__device__ __forceinline__ float share_of(float sum, float total) { return total == 0.f ? 0.f : sum / total; }
// Sums of the waves, [32 columns][DH + 4] each, in LDS.
template <int DH> constexpr int join_bytes(int waves = 4) { return waves * 32 * (DH + 4) * (int)sizeof(float); }

// One record of the softmax of a row from NW waves': called by all threads, f(column, d, sum, maximum, total).
template <int DH, int NW, typename F> __device__ __forceinline__ void join_waves(char* lds, const f32x16* acc, float m, float l, int tid, F f) {
    constexpr int W = DH + 4;
    const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    float* out = reinterpret_cast<float*>(lds);
    float* mine = out + (wave * 32 + (lane & 31)) * W;
    __syncthreads();
    put<float, DH>(mine, acc, 1.f, lane);
    if (lane < 32) { mine[DH] = m; mine[DH + 1] = l; }
    __syncthreads();
    for (int idx = tid; idx < 32 * DH; idx += NW * 64) {
        const int c = idx / DH, d = idx % DH;
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < NW; ++w) top = fmaxf(top, out[(w * 32 + c) * W + DH]);
        float x = 0.f, sum = 0.f;
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const float* rec = out + (w * 32 + c) * W;
            const float e = weight_of(rec[DH], top);
            x += counted(rec[d], rec[DH + 1], e);
            sum += rec[DH + 1] * e;
        }
        f(c, d, x, top, sum);
    }
}
// The plain sum of NW waves': called by all threads, f(column, d, sum).
template <int DH, int NW, typename F> __device__ __forceinline__ void add_waves(char* lds, const f32x16* acc, int tid, F f) {
    constexpr int W = DH + 4;
    const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    float* out = reinterpret_cast<float*>(lds);
    __syncthreads();
    put<float, DH>(out + (wave * 32 + (lane & 31)) * W, acc, 1.f, lane);
    __syncthreads();
    for (int idx = tid; idx < 32 * DH; idx += NW * 64) {
        const int c = idx / DH, d = idx % DH;
        float x = 0.f;
#pragma unroll
        for (int w = 0; w < NW; ++w) x += out[(w * 32 + c) * W + d];
        f(c, d, x);
    }
}

// Tiles of two matrices through LDS, two buffers deep: while one tile is used, the next one is on its way, and one
// barrier a tile orders the two.  use(first tile, second tile, first row); ready() waits for what the loop keeps with the first
// tiles on their way, which gains a little in the forward pass and nothing in the backward kernels.  Returns the buffer that no wave reads
// any more.
template <typename T, int DH, typename R, typename F>
__device__ __forceinline__ char* stream(char* lds, const T* A, long lda, const T* B, long ldb, const Tiles& tl, int n, int tid, R ready, F use) {
    using S = Shape<T, DH>;
    constexpr int BYTES = S::KT * S::ROW;
    const Stage<T, DH> fa(lda, tid), fb(ldb, tid);
    const int cnt = tl.count();
    if (cnt > 0) {
        fa.start(lds, A, tl.at(0) * S::KT, n, tid);
        fb.start(lds + BYTES, B, tl.at(0) * S::KT, n, tid);
    }
    ready();
    for (int t = 0; t < cnt; ++t) {
        char* now = lds + (t & 1) * 2 * BYTES;
        char* next = lds + (~t & 1) * 2 * BYTES;
        dma_wait();
        __syncthreads();
        if (t + 1 < cnt) {
            fa.start(next, A, tl.at(t + 1) * S::KT, n, tid);
            fb.start(next + BYTES, B, tl.at(t + 1) * S::KT, n, tid);
        }
        use(now, now + BYTES, tl.at(t) * S::KT);
    }
    return lds + (cnt & 1) * 2 * BYTES;
}
// 32 rows from r0 of a matrix into an LDS tile of this wave alone, which nothing of it reads any more (wave_reads_done()).
template <typename T, int DH> __device__ __forceinline__ void start_wave(char* tile, const T* base, long ld, int r0, int n, int lane) {
    using S = Shape<T, DH>;
    const unsigned to = __builtin_amdgcn_readfirstlane(lds_addr(tile));
    const T* from = settled(base + r0 * ld);
#pragma unroll
    for (int i = 0; i < 32 * S::CHUNKS / 64; ++i) {
        const int pl = i * 64 + lane, r = pl / S::CHUNKS, ch = (pl % S::CHUNKS) ^ S::mix(r);
        dma16(from, (r0 + r < n ? r : n - 1 - r0) * (int)ld * (int)sizeof(T) + ch * 16, to + i * 1024);
    }
}

// ----------------------------------------------------------------------------- forward
// Element d of an output row from its sums, the maximum behind them (base 2) and their total.
template <typename T, int DH>
__device__ __forceinline__ void write_row(const Slide& p, int b, int h, int i, int d, float sum, float top, float total) {
    const float x = share_of(sum, total);
    const long row = ((long)b * p.N + i) * p.Hq + h;
    ((T*)p.o)[row * DH + d] = (T)x;
    if (sizeof(T) == 2 && p.rest) p.rest[row * DH + d] = (int8_t)rest_of(x);
    if (p.lse && d == 0) p.lse[((long)b * p.Hq + h) * p.N + i] = total == 0.f ? INFINITY : top + __log2f(total);
}
// Band: 128 queries of one (sequence, head), each wave 32 of them; key tiles stream through LDS.
// A head of 64 is bound by vector instructions: 96 beside 8 matrix ones to a 32 x 32 tile, 16 of them exponentials at a
// quarter of the rate (all visible: vector pipes busy 75 % of the cycles, matrix cores 42 %; window 145: 67 and 23 %).  Four waves of 32
// queries share each staged tile; with two tiles in LDS at once and the copies behind the barrier the loop does not wait for memory.
template <typename T, int DH, bool CAUSAL, bool FINE>
__device__ __forceinline__ void fwd_band(const Slide& p, char* lds, int q0, int h, int b, int n) {
    using S = Shape<T, DH>;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), hk = h / p.G;
    const int qa = q0 + wave * 32, qi = qa + (lane & 31);
    const T* K = (const T*)p.k + b * p.k_b + hk * p.k_h;
    const T* V = (const T*)p.v + b * p.v_b + hk * p.v_h;
    Kept<T, DH> q;
    q.load((const T*)p.q + b * p.q_b + h * p.q_h + (long)qi * p.q_n, lane >> 5, qi < n);
    const bool elsewhere = !CAUSAL && qa < p.rows && !p.chunks;          // an item of its own does these rows
    const float sc = p.scale * LOG2E;
    const Span sp = keys_of<CAUSAL>(qi, n, p.window, p.sinks);
    const Cover cover = keys_by<CAUSAL>(qa, n, p.window, p.sinks);
    f32x16 acc[DH / 32] = {};
    Softmax sm;
    const auto rescale = [&](float alpha) {
#pragma unroll
        for (int d = 0; d < DH / 32; ++d) acc[d] *= alpha;
    };
    const Tiles tl = key_tiles<CAUSAL>(q0, q0 + TQ - 1, n, p.window, p.sinks, S::KT);
    char* via = stream<T, DH>(lds, K, p.k_n, V, p.v_n, tl, n, tid, [&] { q.settle(); }, [&](const char* Ks, const char* Vs, int k0) {
#pragma unroll
        for (int sub = 0; sub < S::KT; sub += 32) {
            const int ka = k0 + sub;
            const int cov = cover.of(ka);
            if (cov == 0 || elsewhere) continue;
            f32x16 s = product<DH>(Ks, sub, q, lane);
            if (cov == 1) hide(s, sp, ka + 4 * (lane >> 5), ka < p.sinks, -INFINITY);
            sm.step(s, sc, rescale);
            gather<DH, FINE>(acc, Vs, sub, s, lane, T{});
        }
    });
    const float l = sm.total(), m = sm.m == -INFINITY ? -INFINITY : sm.m * sc;
    if (elsewhere) return;
    if (!CAUSAL && qa < p.rows) {
        float* rec = p.ws + ((((long)b * p.Hq + h) * p.rows + qi) * (p.chunks + 1) + p.chunks) * (DH + 4);
        if (qi >= p.N) return;
        put<float, DH>(rec, acc, 1.f, lane);
        if (lane < 32) { rec[DH] = m; rec[DH + 1] = l; }
        return;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const long row = ((long)b * p.N + qa) * p.Hq + h, ld = (long)p.Hq * DH;
    via += wave * 32 * S::ROW;
    put_rows<DH>(via, (T*)p.o + row * DH, ld, p.N - qa, acc, inv, lane);
    if (sizeof(T) == 2 && p.rest) put_rest<DH>(via, p.rest + row * DH, ld, p.N - qa, acc, inv, lane);
    // base-2 logarithm of the row's sum; +inf for a row that sees nothing, so that backward's probabilities are 0
    if (p.lse && lane < 32 && qi < p.N) p.lse[((long)b * p.Hq + h) * p.N + qi] = l == 0.f ? INFINITY : m + __log2f(l);
}
// Far: 32 first queries against every (4 chunks)-th 32 keys behind their band; or, without chunks, against all they see.
template <typename T, int DH, bool FINE>
__device__ __forceinline__ void fwd_far(const Slide& p, char* lds, int x, int h, int b, int n) {
    using S = Shape<T, DH>;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), hk = h / p.G;
    const bool all = !p.chunks;
    const int chunks = all ? 1 : p.chunks, chunk = x % chunks, qa = x / chunks * 32, qi = qa + (lane & 31);
    char* Ks = lds + wave * 2 * 32 * S::ROW;
    char* Vs = Ks + 32 * S::ROW;
    const T* K = (const T*)p.k + b * p.k_b + hk * p.k_h;
    const T* V = (const T*)p.v + b * p.v_b + hk * p.v_h;
    const bool mine = qi < n && (all || qi < p.sinks);
    Kept<T, DH> q;
    q.load((const T*)p.q + b * p.q_b + h * p.q_h + (long)qi * p.q_n, lane >> 5, mine);
    const float sc = p.scale * LOG2E;
    const Cover cover = keys_by<false>(qa, n, p.window, p.sinks);
    const Span sp = all ? keys_of<false>(qi, n, p.window, p.sinks) : Span{0, mine ? n : 0, 0};
    f32x16 acc[DH / 32] = {};
    Softmax sm;
    const int q0 = qa / TQ * TQ;
    const Tiles tl = key_tiles<false>(q0, q0 + TQ - 1, n, p.window, p.sinks, S::KT);
    const int from = all ? 0 : (tl.hi > tl.first ? tl.hi : tl.first) * S::KT;
    for (int k0 = from + (chunk * 4 + wave) * 32; k0 < n && qa < n; k0 += chunks * 4 * 32) {
        if (all && cover.of(k0) == 0) continue;
        start_wave<T, DH>(Ks, K, p.k_n, k0, n, lane);
        start_wave<T, DH>(Vs, V, p.v_n, k0, n, lane);
        dma_wait();
        wave_lds_fence();
        f32x16 s = product<DH>(Ks, 0, q, lane);
        hide(s, sp, k0 + 4 * (lane >> 5), k0 < p.sinks, -INFINITY);
        sm.step(s, sc, [&](float alpha) {
#pragma unroll
            for (int d = 0; d < DH / 32; ++d) acc[d] *= alpha;
        });
        gather<DH, FINE>(acc, Vs, 0, s, lane, T{});
        wave_reads_done();
    }
    const float l = sm.total(), m = sm.m == -INFINITY ? -INFINITY : sm.m * sc;
    float* base = p.ws + ((((long)b * p.Hq + h) * p.rows + qa) * (chunks + 1) + chunk) * (DH + 4);
    join_waves<DH, 4>(lds, acc, m, l, tid, [&](int c, int d, float sum, float top, float total) {
        if (all) {
            if (qa + c < p.N) write_row<T, DH>(p, b, h, qa + c, d, sum, top, total);
            return;
        }
        float* rec = base + (long)c * (chunks + 1) * (DH + 4);
        rec[d] = sum;
        if (d == 0) { rec[DH] = top; rec[DH + 1] = total; }
    });
}
template <typename T, int DH, bool CAUSAL, bool FINE>
__global__ __launch_bounds__(256, 2) void slide_fwd_kernel(Slide p) {
    extern __shared__ __align__(16) char lds[];
    const Item it = item_of(p, p.Hq, (p.N + TQ - 1) / TQ);
    if (it.none) return;
    const int n = length_of(p, it.b);
    if constexpr (!CAUSAL)
        if (it.far) return fwd_far<T, DH, FINE>(p, lds, it.x, it.h, it.b, n);
    fwd_band<T, DH, CAUSAL, FINE>(p, lds, it.x * TQ, it.h, it.b, n);
}
// One softmax from `count` records of `width` numbers, as element d sees it: several records are in flight at a time.
template <int DH> struct Joined { float x, top, sum; };
template <int DH> __device__ __forceinline__ Joined<DH> join_records(const float* rec, int count, int width, int d) {
    constexpr int U = 8;
    Joined<DH> j{0.f, -INFINITY, 0.f};
    for (int s0 = 0; s0 < count; s0 += U) {
        float m[U], l[U], v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const float* r = rec + (long)least(s0 + u, count - 1) * width;
            const bool is = s0 + u < count;
            m[u] = is ? r[DH] : -INFINITY;
            l[u] = is ? r[DH + 1] : 0.f;
            v[u] = is ? r[d] : 0.f;
        }
        float t = j.top;
#pragma unroll
        for (int u = 0; u < U; ++u) t = fmaxf(t, m[u]);
        const float a = weight_of(j.top, t);
        j.x *= a;
        j.sum *= a;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const float e = weight_of(m[u], t);
            j.x += counted(v[u], l[u], e);
            j.sum += l[u] * e;
        }
        j.top = t;
    }
    return j;
}
// The records of the first rows become outputs.
template <typename T, int DH> __global__ __launch_bounds__(DH < 64 ? 64 : DH) void slide_fwd_join_kernel(Slide p) {
    const int i = blockIdx.x, h = blockIdx.y, b = blockIdx.z, d = threadIdx.x;
    if (d >= DH) return;
    const float* rec = p.ws + (((long)b * p.Hq + h) * p.rows + i) * (p.chunks + 1) * (DH + 4);
    const Joined<DH> j = join_records<DH>(rec, p.chunks + 1, DH + 4, d);
    write_row<T, DH>(p, b, h, i, d, j.x, j.top, j.sum);
}

// ----------------------------------------------------------------------------- backward
// Register r of a score tile belongs to row 8 (r / 4) + r % 4 (+ 4 in the upper half of the wave): the rows' numbers in
// that order.
__device__ __forceinline__ f32x16 rows_of(const float* x, int r0) {
    f32x16 y;
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
        const f32x4 z = *reinterpret_cast<const f32x4*>(x + r0 + 2 * r);
        y[r] = z[0]; y[r + 1] = z[1]; y[r + 2] = z[2]; y[r + 3] = z[3];
    }
    return y;
}
// delta = -dO . o of a kept row, whose elements begin at `at` of o; o with what its rounding left, so that this is not multiplied
// by the cancellation in dP - delta.
template <int DH> __device__ __forceinline__ float delta_of(const Kept<bf16_t, DH>& d_o, const Slide& p, long at, int h, bool ok) {
    float s = 0.f;
#pragma unroll
    for (int c = 0; c < DH / 16; ++c) {
        u32x4 x = {0, 0, 0, 0};
        u32x2 y = {0, 0};
        if (ok) {
            x = *reinterpret_cast<const u32x4*>((const bf16_t*)p.o + at + 16 * c + 8 * h);
            y = *reinterpret_cast<const u32x2*>(p.rest + at + 16 * c + 8 * h);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const unsigned high = e & 1 ? x[e >> 1] & 0xFFFF0000u : x[e >> 1] << 16;
            const int low = ((int)(y[e >> 2] << (24 - 8 * (e & 3))) >> 24) * 256;
            s += (float)d_o.f[c][e] * __uint_as_float(high + (unsigned)low);
        }
    }
    return -(s + __shfl_xor(s, 32, 64));
}
template <int DH> __device__ __forceinline__ float delta_of(const Kept<float, DH>& d_o, const Slide& p, long at, int h, bool ok) {
    const float* o = (const float*)p.o + at;
    float s = 0.f;
#pragma unroll
    for (int t = 0; t < DH / 8; ++t) {
        f32x4 x = {0.f, 0.f, 0.f, 0.f};
        if (ok) x = *reinterpret_cast<const f32x4*>(o + h * (DH / 2) + 4 * t);
#pragma unroll
        for (int e = 0; e < 4; ++e) s += d_o.f[4 * t + e] * x[e];
    }
    return -(s + __shfl_xor(s, 32, 64));
}
// The deltas alone, for a call that wants no dQ (whose kernel leaves them behind otherwise).
template <typename T, int DH> __global__ __launch_bounds__(256) void slide_delta_kernel(Slide p) {
    const int lane = threadIdx.x & 63, h = blockIdx.y, b = blockIdx.z, i = blockIdx.x * TQ + (threadIdx.x >> 6) * 32 + (lane & 31);
    const bool ok = i < length_of(p, b);
    Kept<T, DH> d_o;
    d_o.load((const T*)p.d_o + b * p.do_b + h * p.do_h + (long)i * p.do_n, lane >> 5, ok);
    const float d = delta_of<DH>(d_o, p, (((long)b * p.N + i) * p.Hq + h) * DH, lane >> 5, ok);
    if (i < p.N && lane < 32) p.delta[((long)b * p.Hq + h) * p.N + i] = d;
}

// dQ of a band: as the forward pass, with a second product of the same shape for dP and the deltas on the way (a kernel of its
// own for them takes 18 us, beside 143 of the whole backward pass of 8 images of window 145).  All visible: matrix cores busy 51 % of the
// cycles, vector pipes 62 %.
template <typename T, int DH, bool CAUSAL, bool FINE>
__device__ __forceinline__ void dq_band(const Slide& p, char* lds, int q0, int h, int b, int n) {
    using S = Shape<T, DH>;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), hk = h / p.G;
    const int qa = q0 + wave * 32, qi = qa + (lane & 31);
    const T* K = (const T*)p.k + b * p.k_b + hk * p.k_h;
    const T* V = (const T*)p.v + b * p.v_b + hk * p.v_h;
    Kept<T, DH> q, d_o;
    q.load((const T*)p.q + b * p.q_b + h * p.q_h + (long)qi * p.q_n, lane >> 5, qi < n);
    d_o.load((const T*)p.d_o + b * p.do_b + h * p.do_h + (long)qi * p.do_n, lane >> 5, qi < n);
    const long st = ((long)b * p.Hq + h) * p.N + qi;
    float lse = qi < n ? p.lse[st] : INFINITY;
    float delta = delta_of<DH>(d_o, p, (((long)b * p.N + qi) * p.Hq + h) * DH, lane >> 5, qi < n);
    if (qi < p.N && lane < 32) p.delta[st] = delta;
    q.settle();
    d_o.settle();
    arrived(lse);
    arrived(delta);
    const bool elsewhere = !CAUSAL && qa < p.rows && !p.chunks;
    const float sc = p.scale * LOG2E;
    const Span sp = keys_of<CAUSAL>(qi, n, p.window, p.sinks);
    const Cover cover = keys_by<CAUSAL>(qa, n, p.window, p.sinks);
    f32x16 acc[DH / 32] = {};
    const Tiles tl = key_tiles<CAUSAL>(q0, q0 + TQ - 1, n, p.window, p.sinks, S::KT);
    char* via = stream<T, DH>(lds, K, p.k_n, V, p.v_n, tl, n, tid, [] {}, [&](const char* Ks, const char* Vs, int k0) {
#pragma unroll
        for (int sub = 0; sub < S::KT; sub += 32) {
            const int ka = k0 + sub;
            const int cov = cover.of(ka);
            if (cov == 0 || elsewhere) continue;
            f32x16 s = product<DH>(Ks, sub, q, lane);
            const f32x16 dp = product<DH>(Vs, sub, d_o, lane);
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], sc, -lse)) * (dp[r] + delta);
            if (cov == 1) hide(s, sp, ka + 4 * (lane >> 5), ka < p.sinks, 0.f);      // of hidden pairs it may be infinite
            gather<DH, FINE>(acc, Ks, sub, s, lane, T{});
        }
    });
    if (elsewhere) return;
    if (CAUSAL || qa >= p.rows)
        put_rows<DH>(via + wave * 32 * S::ROW, (T*)p.dq + b * p.dq_b + (long)qa * p.dq_n + h * p.dq_h, p.dq_n, p.N - qa, acc,
                     qi < n ? score_scale(p, n) : 0.f, lane);
    else if (qi < p.N)
        put<float, DH>(p.ws_q + ((((long)b * p.Hq + h) * p.rows + qi) * (p.chunks + 1) + p.chunks) * DH, acc, 1.f, lane);
}
template <typename T, int DH, bool FINE>
__device__ __forceinline__ void dq_far(const Slide& p, char* lds, int x, int h, int b, int n) {
    using S = Shape<T, DH>;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), hk = h / p.G;
    const bool all = !p.chunks;
    const int chunks = all ? 1 : p.chunks, chunk = x % chunks, qa = x / chunks * 32, qi = qa + (lane & 31);
    char* Ks = lds + wave * 2 * 32 * S::ROW;
    char* Vs = Ks + 32 * S::ROW;
    const T* K = (const T*)p.k + b * p.k_b + hk * p.k_h;
    const T* V = (const T*)p.v + b * p.v_b + hk * p.v_h;
    const bool mine = qi < n && (all || qi < p.sinks);
    Kept<T, DH> q, d_o;
    q.load((const T*)p.q + b * p.q_b + h * p.q_h + (long)qi * p.q_n, lane >> 5, mine);
    d_o.load((const T*)p.d_o + b * p.do_b + h * p.do_h + (long)qi * p.do_n, lane >> 5, mine);
    const long st = ((long)b * p.Hq + h) * p.N + qi;
    const float lse = mine ? p.lse[st] : INFINITY;                       // not mine: probabilities of 0
    const float delta = delta_of<DH>(d_o, p, (((long)b * p.N + qi) * p.Hq + h) * DH, lane >> 5, mine);
    const float sc = p.scale * LOG2E;
    const Cover cover = keys_by<false>(qa, n, p.window, p.sinks);
    const Span sp = all ? keys_of<false>(qi, n, p.window, p.sinks) : Span{0, n, 0};
    f32x16 acc[DH / 32] = {};
    const int q0 = qa / TQ * TQ;
    const Tiles tl = key_tiles<false>(q0, q0 + TQ - 1, n, p.window, p.sinks, S::KT);
    const int from = all ? 0 : (tl.hi > tl.first ? tl.hi : tl.first) * S::KT;
    for (int k0 = from + (chunk * 4 + wave) * 32; k0 < n && qa < n; k0 += chunks * 4 * 32) {
        if (all && cover.of(k0) == 0) continue;
        start_wave<T, DH>(Ks, K, p.k_n, k0, n, lane);
        start_wave<T, DH>(Vs, V, p.v_n, k0, n, lane);
        dma_wait();
        wave_lds_fence();
        f32x16 s = product<DH>(Ks, 0, q, lane);
        const f32x16 dp = product<DH>(Vs, 0, d_o, lane);
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], sc, -lse)) * (dp[r] + delta);
        hide(s, sp, k0 + 4 * (lane >> 5), k0 < p.sinks, 0.f);
        gather<DH, FINE>(acc, Ks, 0, s, lane, T{});
        wave_reads_done();
    }
    add_waves<DH, 4>(lds, acc, tid, [&](int c, int d, float sum) {
        const int i = qa + c;
        if (!all) p.ws_q[((((long)b * p.Hq + h) * p.rows + i) * (chunks + 1) + chunk) * DH + d] = sum;
        else if (i < p.N) ((T*)p.dq)[b * p.dq_b + (long)i * p.dq_n + h * p.dq_h + d] = (T)(i < n ? sum * score_scale(p, n) : 0.f);
    });
}
template <typename T, int DH, bool CAUSAL, bool FINE>
__global__ __launch_bounds__(256, sizeof(T) == 2 ? 2 : 1) void slide_dq_kernel(Slide p) {
    extern __shared__ __align__(16) char lds[];
    const Item it = item_of(p, p.Hq, (p.N + TQ - 1) / TQ);
    if (it.none) return;
    const int n = length_of(p, it.b);
    if constexpr (!CAUSAL)
        if (it.far) return dq_far<T, DH, FINE>(p, lds, it.x, it.h, it.b, n);
    dq_band<T, DH, CAUSAL, FINE>(p, lds, it.x * TQ, it.h, it.b, n);
}

// 32 x 32 scores, their probabilities and score gradients, and what they add to dV and dK: rows of the tile are queries,
// columns keys; lse, delta: the rows' (the second product starts from the negative delta).  x0: the query of the tile's
// first row for this lane's half, for `masked` tiles.
template <typename T, int DH, bool FINE, typename K>
__device__ __forceinline__ void dkv_tile(const char* Qs, const char* Os, const float* lse, const float* delta, int sub,
                                         const K& k, const K& v, f32x16* dk, f32x16* dv, float sc, int lane,
                                         bool masked, const Span& sp, int x0, bool first) {
    const int r0 = sub + 4 * (lane >> 5);
    f32x16 s = product<DH>(Qs, sub, k, lane);
    f32x16 dp = product<DH>(Os, sub, v, lane, rows_of(delta, r0));
    const f32x16 ls = rows_of(lse, r0);
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], sc, -ls[r]));
    if (masked) hide(s, sp, x0, first, 0.f);
#pragma unroll
    for (int r = 0; r < 16; ++r) dp[r] *= s[r];
    gather<DH, FINE>(dv, Os, sub, s, lane, T{});
    gather<DH, FINE>(dk, Qs, sub, dp, lane, T{});
}
// How a workgroup of the dK / dV kernel is laid out: NW waves, 32 KG keys; wave w keeps keys 32 (w % KG) and takes every
// (NW / KG)-th 32 queries, and the parts are added at the end.  Four waves of 32 keys each where there are enough of them;
// bands of 64 keys where heads are few; and for bf16 heads of 128, whose four operands and sums of a wave leave room for
// one wave a SIMD only, eight waves with K and V in LDS, two to a SIMD (16384 causal tokens, 2 key heads, window 1024: 164 us, with four
// waves 208).  Without a causal mask the eight waves' kernel keeps 13 registers of a lane in scratch memory and four waves would do (4 x 2305 x
// 8 heads, window 145: 85 us and 75).
template <typename T, int DH, int NW, int KG> struct Layout {
    using S = Shape<T, DH>;
    static constexpr bool IN_LDS = NW == 8;
    using Keep = typename std::conditional<IN_LDS, KeptInLds<T, DH>, Kept<T, DH>>::type;
    static constexpr int PARTS = NW / KG, NT = NW * 64;
    static constexpr int TILE = S::KT * S::ROW, BUF = 2 * TILE + 2 * S::KT * 4;      // Q, dO, lse, delta
    static constexpr int WAVE = 2 * 32 * S::ROW + 256;                               // the same for 32 queries of one wave
    static constexpr int KEEP = IN_LDS ? 32 * KG * S::ROW : 0, KEEP_FAR = IN_LDS ? 32 * S::ROW : 0;      // of K, of V
    static constexpr int MEET = KG * 32 * (DH + 4) * 4;
    static constexpr int most(int a, int b) { return a > b ? a : b; }
    static constexpr int bytes(bool far) {
        const int band = most(2 * BUF + 2 * KEEP, PARTS > 1 ? MEET : 0);
        return far ? most(band, most(NW * WAVE + 2 * KEEP_FAR, join_bytes<DH>(NW))) : band;
    }
};
// Rows of K or V into an LDS tile that stays, zeros from `end` on.
template <typename T, int DH, int NT> __device__ __forceinline__ void keep_rows(char* tile, const T* base, long ld, int r0, int rows, int end, int tid) {
    using S = Shape<T, DH>;
    for (int idx = tid; idx < rows * S::CHUNKS; idx += NT) {
        const int r = idx / S::CHUNKS, ch = idx % S::CHUNKS;
        u32x4 x = {0, 0, 0, 0};
        if (r0 + r < end) x = *reinterpret_cast<const u32x4*>(base + (long)(r0 + r) * ld + ch * (16 / (int)sizeof(T)));
        *reinterpret_cast<u32x4*>(tile + S::at(r, ch)) = x;
    }
}
// Band: the queries of every head that shares the keys stream through LDS, so that dK and dV are sums of one workgroup and need no
// atomics.  All visible, heads of 64: matrix cores busy 48 % of the cycles, vector pipes 42 %, LDS 37 %: four products read a tile in two
// orders, and the registers of two sums leave two waves a SIMD to hide one in the other.
template <typename T, int DH, bool CAUSAL, int NW, int KG, bool FINE>
__device__ __forceinline__ void dkv_band(const Slide& p, char* lds, int k0, int share, int hk, int b, int n) {
    using S = Shape<T, DH>;
    using L = Layout<T, DH, NW, KG>;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int ka = k0 + wave % KG * 32, kj = ka + (lane & 31), part = wave / KG;
    const T* K = (const T*)p.k + b * p.k_b + hk * p.k_h;
    const T* V = (const T*)p.v + b * p.v_b + hk * p.v_h;
    typename L::Keep k, v;
    if constexpr (L::IN_LDS) {
        char* keep = lds + 2 * L::BUF;
        keep_rows<T, DH, L::NT>(keep, K, p.k_n, k0, 32 * KG, n, tid);
        keep_rows<T, DH, L::NT>(keep + L::KEEP, V, p.v_n, k0, 32 * KG, n, tid);
        k.rows = keep + wave % KG * 32 * S::ROW;
        v.rows = k.rows + L::KEEP;
    } else {
        k.load(K + (long)kj * p.k_n, lane >> 5, kj < n);
        v.load(V + (long)kj * p.v_n, lane >> 5, kj < n);
        k.settle();
        v.settle();
    }
    const float sc = p.scale * LOG2E;
    f32x16 dk[DH / 32] = {}, dv[DH / 32] = {};
    const Tiles tl = query_tiles<CAUSAL>(k0, k0 + 32 * KG - 1, n, p.window, p.sinks, S::KT);
    const int per = tl.count();
    int cnt = per * p.G, next_g = 0, next_t = 0;                         // this share's turns, its first one's head and tile
    if (p.shares > 1 && cnt > 0) {
        const int from = (int)((long)cnt * share / p.shares);
        cnt = (int)((long)cnt * (share + 1) / p.shares) - from;
        next_g = from / per;
        next_t = from - next_g * per;
    }
    int tt = next_t;
    const Span sp = queries_of<CAUSAL>(kj, n, p.window, p.sinks);
    const Cover cover = queries_by<CAUSAL>(ka, n, p.window, p.sinks);
    const bool elsewhere = ka < p.rows && !p.chunks;
    const Stage<T, DH, L::NT> fq(p.q_n, tid), fo(p.do_n, tid);
    const auto start = [&](char* buf) {                 // the tiles in order, head after head
        const int h = hk * p.G + next_g, q0 = tl.at(next_t) * S::KT;
        fq.start(buf, (const T*)p.q + b * p.q_b + h * p.q_h, q0, n, tid);
        fo.start(buf + L::TILE, (const T*)p.d_o + b * p.do_b + h * p.do_h, q0, n, tid);
        if (wave < 2 * S::KT / 64) {                    // the rows' lse, delta: rows behind the sequence are masked
            const int x = wave * 64 + lane, i = q0 + x % S::KT;
            const float* from = (x < S::KT ? p.lse : p.delta) + ((long)b * p.Hq + h) * p.N + (i < n ? i : n - 1);
            dma4(from, __builtin_amdgcn_readfirstlane(lds_addr(buf + 2 * L::TILE) + wave * 256));
        }
        if (++next_t == per) { next_t = 0; ++next_g; }
    };
    if (cnt > 0) start(lds);
    for (int t = 0; t < cnt; ++t, tt = tt + 1 == per ? 0 : tt + 1) {
        const char* now = lds + (t & 1) * L::BUF;
        dma_wait();
        __syncthreads();
        if (t + 1 < cnt) start(lds + (~t & 1) * L::BUF);
        const int q0 = tl.at(tt) * S::KT;
        const float* Ls = reinterpret_cast<const float*>(now + 2 * L::TILE);
#pragma unroll
        for (int sub = 0; sub < S::KT; sub += 32) {
            if (L::PARTS == 2 && (((S::KT > 32 ? sub / 32 : t) + part) & 1)) continue;
            const int qa = q0 + sub;
            const int cov = cover.of(qa);
            if (cov == 0 || elsewhere) continue;
            const int x0 = qa + 4 * (lane >> 5);
            const bool first = !CAUSAL && qa < p.sinks;
            dkv_tile<T, DH, FINE>(now, now + L::TILE, Ls, Ls + S::KT, sub, k, v, dk, dv, sc, lane, cov == 1, sp, x0, first);
        }
    }
    if constexpr (L::PARTS == 2) {
        float* at = reinterpret_cast<float*>(lds) + (wave % KG * 32 + (lane & 31)) * (DH + 4);
        const auto meet = [&](f32x16* acc) {
            __syncthreads();
            if (part) put<float, DH>(at, acc, 1.f, lane);
            __syncthreads();
            if (part) return;
#pragma unroll
            for (int d = 0; d < DH / 32; ++d)
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[d][r] += at[32 * d + 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3)];
        };
        meet(dk);
        meet(dv);
        if (part) return;
    }
    if (elsewhere) return;
    if (ka < p.rows || p.shares > 1) {
        if (kj >= p.N) return;
        float* rec = p.shares > 1 ? p.ws_b + ((((long)b * p.Hkv + hk) * p.N + kj) * p.shares + share) * (2 * DH)
                                  : p.ws + ((((long)b * p.Hkv + hk) * p.rows + kj) * (p.chunks + 1) + p.chunks) * (2 * DH);
        put<float, DH>(rec, dk, 1.f, lane);
        put<float, DH>(rec + DH, dv, 1.f, lane);
    } else {
        T* K_to = (T*)p.dk + b * p.dk_b + hk * p.dk_h;
        T* V_to = (T*)p.dv + b * p.dv_b + hk * p.dv_h;
        const float by_k = kj < n ? score_scale(p, n) : 0.f, by_v = kj < n ? 1.f : 0.f;
        if constexpr (L::PARTS == 1) {
            char* via = lds + (cnt & 1) * L::BUF + wave * 32 * S::ROW;                  // no wave reads this buffer any more
            put_rows<DH>(via, K_to + (long)ka * p.dk_n, p.dk_n, p.N - ka, dk, by_k, lane);
            put_rows<DH>(via, V_to + (long)ka * p.dv_n, p.dv_n, p.N - ka, dv, by_v, lane);
        } else if (kj < p.N) {          // half of the waves: the other way gained nothing here
            put<T, DH>(K_to + (long)kj * p.dk_n, dk, by_k, lane);
            put<T, DH>(V_to + (long)kj * p.dv_n, dv, by_v, lane);
        }
    }
}
// Far: 32 first keys against every (NW chunks)-th 32 queries behind their band, of every head that shares them.
template <typename T, int DH, bool CAUSAL, int NW, int KG, bool FINE>
__device__ __forceinline__ void dkv_far(const Slide& p, char* lds, int x, int hk, int b, int n) {
    using S = Shape<T, DH>;
    using L = Layout<T, DH, NW, KG>;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const bool all = !p.chunks;
    const int chunks = all ? 1 : p.chunks, chunk = x % chunks, ka = x / chunks * 32, kj = ka + (lane & 31);
    char* Qs = lds + wave * L::WAVE;
    char* Os = Qs + 32 * S::ROW;
    float* Ls = reinterpret_cast<float*>(Os + 32 * S::ROW);             // [32] lse, [32] delta
    const int last = all ? n : least(n, p.sinks);
    const bool mine = kj < last;
    const T* K = (const T*)p.k + b * p.k_b + hk * p.k_h;
    const T* V = (const T*)p.v + b * p.v_b + hk * p.v_h;
    typename L::Keep k, v;
    if constexpr (L::IN_LDS) {
        char* keep = lds + NW * L::WAVE;
        keep_rows<T, DH, L::NT>(keep, K, p.k_n, ka, 32, last, tid);
        keep_rows<T, DH, L::NT>(keep + L::KEEP_FAR, V, p.v_n, ka, 32, last, tid);
        k.rows = keep;
        v.rows = keep + L::KEEP_FAR;
        __syncthreads();
    } else {
        k.load(K + (long)kj * p.k_n, lane >> 5, mine);
        v.load(V + (long)kj * p.v_n, lane >> 5, mine);
    }
    const float sc = p.scale * LOG2E;
    f32x16 dk[DH / 32] = {}, dv[DH / 32] = {};
    const int k0 = ka / (32 * KG) * (32 * KG);
    const Tiles tl = query_tiles<CAUSAL>(k0, k0 + 32 * KG - 1, n, p.window, p.sinks, S::KT);
    const int from = all ? 0 : (tl.hi > tl.first ? tl.hi : tl.first) * S::KT;
    const Cover cover = queries_by<CAUSAL>(ka, n, p.window, p.sinks);
    const Span sp = all ? queries_of<CAUSAL>(kj, n, p.window, p.sinks) : Span{0, mine ? n : 0, 0};
    const int per = ka < n && from < n ? (n - from + 31) / 32 : 0;
    for (int t = chunk * NW + wave; t < per * p.G; t += chunks * NW) {
        const int h = hk * p.G + t / per, q0 = from + t % per * 32;
        if (all && cover.of(q0) == 0) continue;
        const long st = ((long)b * p.Hq + h) * p.N + q0;
        start_wave<T, DH>(Qs, (const T*)p.q + b * p.q_b + h * p.q_h, p.q_n, q0, n, lane);
        start_wave<T, DH>(Os, (const T*)p.d_o + b * p.do_b + h * p.do_h, p.do_n, q0, n, lane);
        const int r = lane & 31;
        Ls[lane] = (lane < 32 ? p.lse : p.delta)[st + (q0 + r < n ? r : n - 1 - q0)];
        dma_wait();
        wave_lds_fence();
        dkv_tile<T, DH, FINE>(Qs, Os, Ls, Ls + 32, 0, k, v, dk, dv, sc, lane, true, sp, q0 + 4 * (lane >> 5), !CAUSAL && q0 < p.sinks);
        wave_reads_done();
    }
    const auto leave = [&](f32x16* acc, bool values) {
        add_waves<DH, NW>(lds, acc, tid, [&](int c, int d, float sum) {
            const int j = ka + c;
            if (!all) {
                p.ws[((((long)b * p.Hkv + hk) * p.rows + j) * (chunks + 1) + chunk) * (2 * DH) + (values ? DH : 0) + d] = sum;
            } else if (j < p.N) {
                if (values) ((T*)p.dv)[b * p.dv_b + (long)j * p.dv_n + hk * p.dv_h + d] = (T)(j < n ? sum : 0.f);
                else ((T*)p.dk)[b * p.dk_b + (long)j * p.dk_n + hk * p.dk_h + d] = (T)(j < n ? sum * score_scale(p, n) : 0.f);
            }
        });
    };
    leave(dk, false);
    leave(dv, true);
}
template <typename T, int DH, bool CAUSAL, int NW, int KG, bool FINE>
__global__ __launch_bounds__(NW * 64, sizeof(T) == 2 && (DH < 128 || NW == 8) ? 2 : 1) void slide_dkv_kernel(Slide p) {
    extern __shared__ __align__(16) char lds[];
    const Item it = item_of(p, p.Hkv, (p.N + 32 * KG - 1) / (32 * KG) * p.shares);
    if (it.none) return;
    const int n = length_of(p, it.b);
    if (it.far) dkv_far<T, DH, CAUSAL, NW, KG, FINE>(p, lds, it.x, it.h, it.b, n);
    else {
        const int band = p.shares > 1 ? it.x / p.shares : it.x;
        dkv_band<T, DH, CAUSAL, NW, KG, FINE>(p, lds, band * (32 * KG), it.x - band * p.shares, it.h, it.b, n);
    }
}
// Records become gradients.  Of the keys that are first tokens: their far items' and the band's; of all keys, where shares of
// a band were done apart: the shares'.  Of the queries that are first tokens (the workgroups behind `keys` ones): their
// items' and the band's.  NT / DH parts of the workgroup add some of them, each in its order, and then their sums in theirs.
template <typename T, int DH, int NT> __global__ __launch_bounds__(NT) void slide_bwd_join_kernel(Slide p, int keys, int rows, int k_chunks, int q_chunks) {
    constexpr int SHARES = NT / DH;
    __shared__ float part[2][NT];
    const bool key = (int)blockIdx.x < keys;
    const int id = key ? blockIdx.x : blockIdx.x - keys, heads = key ? p.Hkv : p.Hq;
    const int i = id / heads, h = id % heads, b = blockIdx.y, d = threadIdx.x % DH, share = threadIdx.x / DH;
    const int width = key ? 2 * DH : DH, chunks = key ? k_chunks : q_chunks;
    if (key && !chunks && i < rows) return;                   // done by items of their own
    const bool split = key && p.shares > 1;
    float x = 0.f, y = 0.f;
    const auto add = [&](const float* rec, int count) {
#pragma unroll 4
        for (int s = share; s < count; s += SHARES) {
            x += rec[(long)s * width + d];
            if (key) y += rec[(long)s * width + DH + d];
        }
    };
    if (i < rows) add((key ? p.ws : p.ws_q) + (((long)b * heads + h) * rows + i) * (chunks + 1) * width, chunks + !split);
    if (split) add(p.ws_b + (((long)b * heads + h) * p.N + i) * p.shares * width, p.shares);
    part[0][threadIdx.x] = x;
    part[1][threadIdx.x] = y;
    __syncthreads();
    if (share) return;
#pragma unroll
    for (int s = 1; s < SHARES; ++s) { x += part[0][s * DH + d]; y += part[1][s * DH + d]; }
    const int n = length_of(p, b);
    const bool there = i < n;
    if (key) {
        ((T*)p.dk)[b * p.dk_b + (long)i * p.dk_n + h * p.dk_h + d] = (T)(there ? x * score_scale(p, n) : 0.f);
        ((T*)p.dv)[b * p.dv_b + (long)i * p.dv_n + h * p.dv_h + d] = (T)(there ? y : 0.f);
    } else {
        ((T*)p.dq)[b * p.dq_b + (long)i * p.dq_n + h * p.dq_h + d] = (T)(there ? x * score_scale(p, n) : 0.f);
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
// The heads that share a key head are the 32 MFMA columns.  Memory-bound, 5.9 TB/s with 32 streams of 8192 keys (8 key heads of 128:
// 184 us; a large copy reaches 5.0, which writes as much as it reads, a library's sum 4.0): each of NW waves stages its own 32 keys at a time (no
// barrier in the loop) and keeps a softmax of its own; the waves are joined through LDS, the splits through the workspace:
// [B, Hq, splits] records of DH sums, a maximum (scaled, base 2) and a sum.
// Probabilities go into their product as two bf16 numbers each, since matrix cores wait for memory here: an output is off by its own
// rounding alone, 0.00165 of the norm, where one number each leaves 0.0023 (32 streams: 184 us both; what one workgroup alone does with 1000
// keys of 64 elements: 7.6 and 8.9 us).
template <typename T, int DH, int NW>
__global__ __launch_bounds__(NW * 64, 1) void slide_decode_kernel(Decode p) {
    using S = Shape<T, DH>;
    extern __shared__ __align__(16) char lds[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
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
    for (int t = split * NW + wave; t < tf + tw; t += p.splits * NW) {
        const int k0 = t < tf ? t * 32 : back + (t - tf) * 32;
        const int end = t < tf ? f : n;
        Fetch<T, DH> fk, fv;
        fk.load(K, p.k_n, k0, end, lane);
        fv.load(V, p.v_n, k0, end, lane);
        fk.store(Ks, lane);
        fv.store(Vs, lane);
        wave_lds_fence();
        f32x16 s = product<DH>(Ks, 0, q, lane);
        if (k0 + 32 > end) hide(s, Span{0, end, 0}, k0 + 4 * (lane >> 5), false, -INFINITY);
        sm.step(s, sc, [&](float alpha) {
#pragma unroll
            for (int d = 0; d < DH / 32; ++d) acc[d] *= alpha;
        });
        gather<DH, true>(acc, Vs, 0, s, lane, T{});
        wave_lds_fence();
    }
    const float l = sm.total(), m = sm.m == -INFINITY ? -INFINITY : sm.m * sc;
    join_waves<DH, NW>(lds, acc, m, l, tid, [&](int c, int d, float x, float top, float sum) {
        if (g0 + c >= p.G) return;
        const long row = (long)b * p.Hq + hk * p.G + g0 + c;
        if (p.splits == 1) {
            ((T*)p.o)[row * DH + d] = (T)share_of(x, sum);
        } else {
            float* rec = p.ws + (row * p.splits + split) * (DH + 2);
            rec[d] = x;
            if (d == 0) { rec[DH] = top; rec[DH + 1] = sum; }
        }
    });
}
template <typename T, int DH> __global__ __launch_bounds__(DH < 64 ? 64 : DH) void slide_join_kernel(Decode p) {
    const long row = blockIdx.x;
    const int d = threadIdx.x;
    if (d >= DH) return;
    const Joined<DH> j = join_records<DH>(p.ws + row * p.splits * (DH + 2), p.splits, DH + 2, d);
    ((T*)p.o)[row * DH + d] = (T)share_of(j.x, j.sum);
}

// ----------------------------------------------------------------------------- host side
template <typename K> int allow_lds(K kernel, int bytes) {
    if (bytes <= 64 * 1024) return 0;
    return (int)hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
}
constexpr int dkv_waves(bool bf16, int dh) { return bf16 && dh == 128 ? 8 : 4; }
// Items of the first tokens: rows (a multiple of 32; 0: none needed), chunks of far items for each 32 of them, floats of
// workspace for their records.  One item for all (no records, no second launch) while it ends before the bands do, which
// its turns, of a microsecond or so each, decide: up to 24 of its waves where there are four bands a CU and more (2305 tokens,
// 8 sequences of 12 heads: forward 52 us, with chunks 57; backward 143, with chunks 156), up to 12 with fewer bands (577
// tokens, 6 of 8 heads: backward 36 us, with chunks 39; 2305 tokens, one of 12 heads: 57 us, with chunks 38, and four, just below the
// border: 83 and 94; 16384 causal tokens, 2 key heads of 4 queries each: 659 us, with chunks 276).  Else a chunk gives each of its
// waves about 4 far tiles (that backward: 2 tiles 281 us, 4 276, 8 282), and fewer chunks do where there are items enough without them.
struct Records { int rows, chunks; long floats; };
Records records_of(int B, int N, int heads, int G, int width, int window, int sinks, int waves) {
    Records r{0, 0, 0};
    if (sinks <= 0 || window >= N) return r;
    r.rows = (sinks + 31) / 32 * 32;
    const long tiles = (long)G * ((N + 31) / 32);
    const long bands = (long)B * heads * ((N + TQ - 1) / TQ);
    if (tiles <= (bands >= 1024 ? 24 : 12) * waves) return r;
    const long items = (long)B * heads * (r.rows / 32), most = (2048 + items - 1) / items;
    r.chunks = (int)((tiles + 4 * waves - 1) / (4 * waves));
    if (r.chunks > most) r.chunks = (int)most;
    if (r.chunks > 512) r.chunks = 512;
    r.floats = (long)B * heads * r.rows * (r.chunks + 1) * width;
    return r;
}
// Bands of the dK / dV kernel: 32 `groups` keys, `shares` workgroups each, floats of workspace for their records.  Bands of 64
// keys where there are fewer than two of 128 for each CU (577 tokens, 6 of 4 key heads: 23 us, bands of 128 28; 25 of 6, which is 750 bands:
// 80 us, bands of 128 66), and then as many shares as it takes to fill the chip, of 8 turns and more, behind which the records
// are added (4096 causal tokens, 2 key heads of 4 queries each, 128 elements, window 1024: 65 us, unsplit 135; 1024 tokens of 64: 21 us and 63,
// with shares of 2 turns 24; the 577 tokens with shares of 2 turns 37).  Times with the deltas' kernel.
struct Bands { int groups, shares; long floats; };
Bands bands_of(int B, int N, int Hkv, int G, bool causal, int window, bool bf16, int dh) {
    Bands r{4, 1, 0};
    const bool wide = dkv_waves(bf16, dh) == 8;
    if (!wide && (long)vitk_ceil_div(N, TQ) * Hkv * B < 512) r.groups = 2;
    const long bands = (long)vitk_ceil_div(N, 32 * r.groups) * Hkv * B;
    const long reach = (causal ? window : 2L * window) + 32 * r.groups, turns = G * (((reach < N ? reach : N) + 63) / 64);
    const long some = (wide ? 256 : 512) / bands, least = turns / 8;
    r.shares = (int)(some < least ? some : least);
    if (r.shares < 2) r.shares = 1;
    else r.floats = (long)B * Hkv * N * r.shares * 2 * dh;
    return r;
}
// Window and sinks of N tokens without what they cannot tell apart: all visible is a window of N.
void reach(const vitk_slide_attn* a, int& window, int& sinks) {
    window = a->window < a->N ? a->window : a->N;
    sinks = a->sinks;
    if (sinks >= a->N) window = a->N;
    if (window >= a->N) sinks = 0;
}
unsigned grid_of(Slide& p, int heads, bool far, int rows = TQ, int shares = 1) {
    p.far_items = far ? (p.chunks ? p.chunks : 1) * (p.rows / 32) * heads * p.B : 0;
    const long bands = (long)vitk_ceil_div(p.N, rows) * heads * p.B * shares;
    p.items = (int)(p.far_items + bands);
    return (unsigned)(p.far_items + (bands + 7) / 8 * 8);
}
template <typename T, int DH> constexpr int lds_bytes(bool far) {      // of the forward and the dQ kernel
    const int band = 4 * Shape<T, DH>::KT * Shape<T, DH>::ROW, staged = 4 * 2 * 32 * Shape<T, DH>::ROW;
    const int joined = join_bytes<DH>(), wide = staged > joined ? staged : joined;
    return far && wide > band ? wide : band;
}
template <typename T, int DH, bool CAUSAL, int NW, int KG, bool FINE> int launch_dkv(Slide& p, hipStream_t st) {
    const int bytes = Layout<T, DH, NW, KG>::bytes(p.rows > 0);
    if (int e = allow_lds(slide_dkv_kernel<T, DH, CAUSAL, NW, KG, FINE>, bytes)) return e;
    const unsigned grid = grid_of(p, p.Hkv, p.rows > 0, 32 * KG, p.shares);
    hipLaunchKernelGGL((slide_dkv_kernel<T, DH, CAUSAL, NW, KG, FINE>), dim3(grid), dim3(NW * 64), bytes, st, p);
    VITK_CHECK_LAUNCH();
    return 0;
}
template <typename T, int DH, bool CAUSAL, bool FINE> int run_fwd(Slide p, float* ws, hipStream_t st) {
    if (!CAUSAL) {
        const Records r = records_of(p.B, p.N, p.Hq, 1, DH + 4, p.window, p.sinks, 4);
        p.rows = r.rows; p.chunks = r.chunks; p.ws = ws;
        if (r.floats && !ws) return VITK_ERR_NULL;
    }
    const int bytes = lds_bytes<T, DH>(p.rows > 0);
    if (int e = allow_lds(slide_fwd_kernel<T, DH, CAUSAL, FINE>, bytes)) return e;
    const unsigned grid = grid_of(p, p.Hq, p.rows > 0);
    hipLaunchKernelGGL((slide_fwd_kernel<T, DH, CAUSAL, FINE>), dim3(grid), dim3(256), bytes, st, p);
    VITK_CHECK_LAUNCH();
    if (p.chunks) {
        hipLaunchKernelGGL((slide_fwd_join_kernel<T, DH>), dim3(p.rows < p.N ? p.rows : p.N, p.Hq, p.B), dim3(DH < 64 ? 64 : DH), 0, st, p);
        VITK_CHECK_LAUNCH();
    }
    return 0;
}
template <typename T, int DH, bool CAUSAL, bool FINE> int run_bwd(Slide p, float* ws, hipStream_t st) {
    const Records rk = records_of(p.B, p.N, p.Hkv, p.G, 2 * DH, p.window, p.sinks, dkv_waves(sizeof(T) == 2, DH));
    const Bands bands = bands_of(p.B, p.N, p.Hkv, p.G, CAUSAL, p.window, sizeof(T) == 2, DH);
    const Records rq = CAUSAL ? Records{0, 0, 0} : records_of(p.B, p.N, p.Hq, 1, DH, p.window, p.sinks, 4);
    if (rk.floats + bands.floats + rq.floats && !ws) return VITK_ERR_NULL;
    const int bytes = lds_bytes<T, DH>(rq.rows > 0);
    if (int e = allow_lds(slide_dq_kernel<T, DH, CAUSAL, FINE>, bytes)) return e;
    p.ws = ws;
    p.ws_b = ws + rk.floats;
    p.ws_q = p.ws_b + bands.floats;
    p.shares = bands.shares;
    if (p.dq) {
        p.rows = rq.rows; p.chunks = rq.chunks;
        const unsigned grid = grid_of(p, p.Hq, rq.rows > 0);
        hipLaunchKernelGGL((slide_dq_kernel<T, DH, CAUSAL, FINE>), dim3(grid), dim3(256), bytes, st, p);
    } else {
        hipLaunchKernelGGL((slide_delta_kernel<T, DH>), dim3(vitk_ceil_div(p.N, TQ), p.Hq, p.B), dim3(256), 0, st, p);
    }
    VITK_CHECK_LAUNCH();
    if (p.dk) {
        p.rows = rk.rows; p.chunks = rk.chunks;
        int e;
        if constexpr (dkv_waves(sizeof(T) == 2, DH) == 8) e = launch_dkv<T, DH, CAUSAL, 8, 4, FINE>(p, st);
        else if (bands.groups == 2) e = launch_dkv<T, DH, CAUSAL, 4, 2, FINE>(p, st);
        else e = launch_dkv<T, DH, CAUSAL, 4, 4, FINE>(p, st);
        if (e) return e;
    }
    const int first = rk.rows < p.N ? rk.rows : p.N;
    const int keys = !p.dk ? 0 : (bands.shares > 1 ? p.N : rk.chunks ? first : 0) * p.Hkv, queries = p.dq && rq.chunks ? first * p.Hq : 0;
    if (keys + queries) {
        // many records of few rows are added by 1024 threads (16384 tokens, 64 chunks: backward 276 us, with 256 threads 282)
        if (bands.shares == 1 && (rk.chunks >= 32 || rq.chunks >= 32))
            hipLaunchKernelGGL((slide_bwd_join_kernel<T, DH, 1024>), dim3(keys + queries, p.B), dim3(1024), 0, st, p, keys, rk.rows, rk.chunks, rq.chunks);
        else
            hipLaunchKernelGGL((slide_bwd_join_kernel<T, DH, 256>), dim3(keys + queries, p.B), dim3(256), 0, st, p, keys, rk.rows, rk.chunks, rq.chunks);
        VITK_CHECK_LAUNCH();
    }
    return 0;
}
// In bf16, probabilities and score gradients go into their products as two numbers each where a window holds few keys: o, dQ, dK and
// dV are then off by their own rounding alone (0.0016 to 0.0017 of their norm), and by 0.0024 with one number each, dQ and dK of rows
// of a few keys by 0.0025 and more: the deltas take over the error of o, which has nothing to average over there.  8 x 2305 x 12 x 64, one
// number and two, whole calls: window 16 forward 33 us and 36, backward 106 and 118; window 33 33 and 35, 102 and 115; window 145 46 and
// 57, 143 and 172.  16384 causal tokens, 8 heads of 2 x 128: window 16 30 and 32, 99 and 109; window 1024 84 and 110, 275 and 354.
// The rule goes by the window: the first rows of a causal sequence and sequences of up to 16 tokens in a longer batch, which see few keys under
// any window, stay at one number.
constexpr int FINE_WINDOW = 16;
template <typename T, int DH, bool CAUSAL> int run_fwd(const Slide& p, float* ws, hipStream_t st) {
    if constexpr (sizeof(T) == 2)
        if (p.window <= FINE_WINDOW) return run_fwd<T, DH, CAUSAL, true>(p, ws, st);
    return run_fwd<T, DH, CAUSAL, false>(p, ws, st);
}
template <typename T, int DH, bool CAUSAL> int run_bwd(const Slide& p, float* ws, hipStream_t st) {
    if constexpr (sizeof(T) == 2)
        if (p.window <= FINE_WINDOW) return run_bwd<T, DH, CAUSAL, true>(p, ws, st);
    return run_bwd<T, DH, CAUSAL, false>(p, ws, st);
}
template <typename T, int DH> int run_decode(const Decode& p, hipStream_t st) {
    constexpr int NW = sizeof(T) == 2 ? 8 : 4;                         // what LDS holds of a head of 128
    constexpr int tiles = NW * 2 * 32 * Shape<T, DH>::ROW, join = join_bytes<DH>(NW), bytes = tiles > join ? tiles : join;
    if (int e = allow_lds(slide_decode_kernel<T, DH, NW>, bytes)) return e;
    hipLaunchKernelGGL((slide_decode_kernel<T, DH, NW>), dim3(p.splits, p.Hkv * ((p.G + 31) / 32), p.B), dim3(NW * 64), bytes, st, p);
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
    if (a->B <= 0 || a->N <= 0 || a->Hq <= 0 || a->Hkv <= 0 || a->Hq % a->Hkv || a->B > 65535 || a->Hq > 32767) return VITK_ERR_SHAPE;
    if (a->N > (1 << 30) || a->window < 0 || a->sinks < 0 || !(a->scale > 0.f && a->scale * LOG2E < INFINITY)) return VITK_ERR_SHAPE;
    const int e = dtype == VITK_BF16 ? 2 : 4;
    if (!aligned(a->q, e, {a->q_b, a->q_n, a->q_h}) || !aligned(a->k, e, {a->k_b, a->k_n, a->k_h}) ||
        !aligned(a->v, e, {a->v_b, a->v_n, a->v_h})) return VITK_ERR_SHAPE;
    p = Slide{};
    p.q = a->q; p.k = a->k; p.v = a->v; p.o = a->o; p.rest = (int8_t*)a->o_rest; p.lse = a->lse; p.lengths = a->lengths;
    p.B = a->B; p.N = a->N; p.Hq = a->Hq; p.Hkv = a->Hkv; p.G = a->Hq / a->Hkv;
    p.q_b = a->q_b; p.q_n = a->q_n; p.q_h = a->q_h;
    p.k_b = a->k_b; p.k_n = a->k_n; p.k_h = a->k_h;
    p.v_b = a->v_b; p.v_n = a->v_n; p.v_h = a->v_h;
    reach(a, p.window, p.sinks);
    p.single = (p.window == 1 && p.sinks == 0) || (p.window == 0 && p.sinks == 1 && a->causal);
    // a tile's rows are addressed with 32 bits from its first one on
    for (long ld : {a->q_n, a->k_n, a->v_n, backward ? a->do_n : 0L})
        if (ld < 0 || ld >= (1L << 23)) return VITK_ERR_SHAPE;
    if ((uintptr_t)a->workspace % 16) return VITK_ERR_SHAPE;
    // items of a launch are counted in 31 bits
    if (((long)a->N / TQ + 2) * a->Hq * a->B > (1L << 30)) return VITK_ERR_SHAPE;
    p.scale = a->scale;
    if (!backward) {
        if (!a->o) return VITK_ERR_NULL;
        return aligned(a->o, e, {}) && aligned(a->o_rest, 1, {}) ? 0 : VITK_ERR_SHAPE;
    }
    if (!a->d_o || !a->lse || !a->delta || !a->dk != !a->dv || !(a->dq || a->dk)) return VITK_ERR_NULL;
    if (!a->o || (dtype == VITK_BF16 && !a->o_rest)) return VITK_ERR_NULL;
    if (!aligned(a->o, e, {}) || !aligned(a->o_rest, 1, {})) return VITK_ERR_SHAPE;
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

extern "C" size_t vitk_slide_attn_workspace(const vitk_slide_attn* a, int dtype, int backward) {
    if (!a || a->B <= 0 || a->N <= 0 || a->Hq <= 0 || a->Hkv <= 0 || a->Hq % a->Hkv || a->dh <= 0) return 0;
    int window, sinks;
    reach(a, window, sinks);
    long n = 0;
    if (!backward) {
        if (!a->causal) n = records_of(a->B, a->N, a->Hq, 1, a->dh + 4, window, sinks, 4).floats;
    } else {
        n = records_of(a->B, a->N, a->Hkv, a->Hq / a->Hkv, 2 * a->dh, window, sinks, dkv_waves(dtype == VITK_BF16, a->dh)).floats;
        n += bands_of(a->B, a->N, a->Hkv, a->Hq / a->Hkv, a->causal, window, dtype == VITK_BF16, a->dh).floats;
        if (!a->causal) n += records_of(a->B, a->N, a->Hq, 1, a->dh, window, sinks, 4).floats;
    }
    return (size_t)n * sizeof(float);
}

extern "C" int vitk_slide_attn_fwd(const vitk_slide_attn* a, int dtype, void* stream) {
    Slide p;
    if (int e = fill(a, dtype, false, p)) return e;
    hipStream_t st = (hipStream_t)stream;
#define FWD(T, DH, C) run_fwd<T, DH, C>(p, a->workspace, st)
    SLIDE_FORMS(FWD);
}

extern "C" int vitk_slide_attn_bwd(const vitk_slide_attn* a, int dtype, void* stream) {
    Slide p;
    if (int e = fill(a, dtype, true, p)) return e;
    hipStream_t st = (hipStream_t)stream;
#define BWD(T, DH, C) run_bwd<T, DH, C>(p, a->workspace, st)
    SLIDE_FORMS(BWD);
}

extern "C" int vitk_slide_decode(const vitk_slide_cache* a, int dtype, void* stream) {
    if (!a || !a->q || !a->k || !a->v || !a->o || !a->lengths) return VITK_ERR_NULL;
    if (dtype != VITK_BF16 && dtype != VITK_F32) return VITK_ERR_DTYPE;
    if (a->dh != 32 && a->dh != 64 && a->dh != 128) return VITK_ERR_UNSUPPORTED;
    if (a->B <= 0 || a->cap <= 0 || a->Hq <= 0 || a->Hkv <= 0 || a->Hq % a->Hkv || a->B > 65535) return VITK_ERR_SHAPE;
    if (a->cap > (1 << 30) || a->window < 0 || a->sinks < 0 || !(a->scale > 0.f && a->scale * LOG2E < INFINITY) || a->splits < 1 || a->splits > 1024) return VITK_ERR_SHAPE;
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
