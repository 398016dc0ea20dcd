// Arguments and row folding shared by the cross-attention kernels (xattn.hip, xattn_step.hip).
#pragma once
#include "attn_tiles.h"
#include <initializer_list>

// include/sarnet.h: sarXattn (kept field for field)
struct sarXattn {
    const void *q, *k, *v, *dout;
    void* out;
    float* lse;
    void *dq, *dk, *dv;
    const int *k_lens, *q_lens;
    void* ws;
    long ws_bytes;
    long q_sb, q_st, q_sh, k_sb, k_st, k_sh, v_sb, v_st, v_sh, o_sb, o_st, o_sh, g_sb, g_st, g_sh;
    int B, Tq, Tk, Hq, Hkv, D;
    float scale;
    int elt_bytes;
};

namespace attn {

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr float NO_MAX = -3.402823e38f; // the running maximum before any key: finite, so that exp2(x - NO_MAX) is a number (0 for x = -inf) without a special case

// The query heads of one key head are folded into the rows: row r = t G + g is token t of query head hkv G + g, so a key / value tile is
// fetched once for all of them, and G tokens of a single-token step share one MFMA tile.
__device__ __forceinline__ int live_keys(const sarXattn& a, int b) { return a.k_lens ? min(max(a.k_lens[b], 0), a.Tk) : a.Tk; }
__device__ __forceinline__ int live_rows(const sarXattn& a, int b) { return (a.q_lens ? min(max(a.q_lens[b], 0), a.Tq) : a.Tq) * (a.Hq / a.Hkv); }

// |scale| log2 e; for a scale of 0 the smallest number, which makes nothing of any finite product and leaves -inf what it is
constexpr float LEAST = 1.401298464324817e-45f;
__device__ __forceinline__ float score_factor(const sarXattn& a) { return fmaxf(fabsf(a.scale) * LOG2E, LEAST); }

// exp2(s f - m), m = the largest s f, rounded: one fma, whose product is exact; the rounding of m comes back as a factor that p and its sum share --
// until m passes LARGE, where the factor itself would do harm: then the product is rounded as m's was, and the difference is exact.  (A branch per
// tile, not a choice per element: 281 against 310 us for the forward of 8 x 1024 x 4096.)
constexpr float LARGE = 1048576.f;
template <int N> __device__ __forceinline__ void exponents(f32x16 (&s)[N], float f, float m, bool large) {
#pragma clang fp contract(off)
    if (large) {
#pragma unroll
        for (int u = 0; u < N; ++u)
#pragma unroll
            for (int i = 0; i < 16; ++i) { const float y = s[u][i] * f; s[u][i] = y - m; }
    } else {
#pragma unroll
        for (int u = 0; u < N; ++u)
#pragma unroll
            for (int i = 0; i < 16; ++i) s[u][i] = fmaf(s[u][i], f, -m);
    }
}
// lse in powers of two for the backward's p = exp2(s f - e).  It is rounded too: past 2^22 by whole units, which decide what p comes out as.  There it is
// moved up by its roundings, so that no p is above 1 and the gradients stay finite.  A row that met no score (lse -inf) gets 0.
// up: p is wanted times 2^up (below 2^22 that costs nothing of e: up is a multiple of its last place).
__device__ __forceinline__ float backward_exponent(float lse, float up = 0.f) {
    const float e = lse * LOG2E, a = fabsf(e), r = e - up;
    return e == -INFINITY ? 0.f : a > 4194304.f ? fmaf(a, 2.384185791015625e-7f, r) : r;
}

// The forward's running reference m of a row's exponents follows the maximum `top` only where that is more than LAG ahead (a row starts with its first
// maximum): most tiles skip the rescaling.  p = 2^(s f - m) is 2^LAG at most, which loses nothing in bf16 and fp32.  fp16 is used in full: m stays BELOW
// the maximum, so that p reaches up to 2^15 and is a normal number down to 2^-26 .. 2^-29 of the largest (a key that takes nearly all of the weight, and
// whose v is 0, leaves the result to the others).  (top - m, not m + LAG: the sum rounds by whole units past 2^24.)
template <typename C> constexpr float lag() { return __is_same(C, _Float16) ? 15.f : 8.f; }
template <typename C> __device__ __forceinline__ float reference(float top) { return __is_same(C, _Float16) && fabsf(top) < LARGE ? top - 12.f : top; }

struct Row { int t, h; };
__device__ __forceinline__ Row row_of(const sarXattn& a, int hkv, int r) {
    const int G = a.Hq / a.Hkv, t = r / G;
    return {t, hkv * G + (r - t * G)};
}
// position of a row's statistics: lse is (B, Hq, Tq)
__device__ __forceinline__ long stat_at(const sarXattn& a, int b, Row w) { return ((long)b * a.Hq + w.h) * a.Tq + w.t; }

// the split form's partial results: O (splits, rows, D) fp32, then m and l (splits, rows); rows = B Hq Tq
__device__ __host__ __forceinline__ long part_floats(long rows, int D, int splits) { return splits * rows * (D + 2); }

// ---- host side: what a call may look like, and how far its key axis is cut
static inline bool bad_shape(const sarXattn* a) {
    if (!a || a->B < 1 || a->Tq < 1 || a->Tk < 0 || a->Hkv < 1 || a->Hq < 1 || a->Hq % a->Hkv || a->D < 8 || a->D > 128 || a->D % 8) return true;
    const long R = (long)a->Tq * (a->Hq / a->Hkv);
    // a launch has fewer than 2^32 threads: 512 for 32 rows at most, 256 for 128 keys
    return R > (1L << 30) || a->Tk > (1 << 30) || (R + 31) / 32 * a->B * a->Hkv > (1L << 23) - 8 || (a->Tk + 127L) / 128 * a->B * a->Hkv > (1L << 24) - 8;
}
static inline bool bad_strides(int elt_bytes, const long* s, int n) {
    for (int i = 0; i < n; ++i)
        if (s[i] < 0 || s[i] > (1L << 40) || s[i] * elt_bytes % 16) return true;
    return false;
}
// a tile's rows are addressed with 32-bit offsets from its first: rows at most 16 MB apart
static inline bool wide_rows(int elt_bytes, std::initializer_list<long> strides) {
    for (long s : strides)
        if (s * elt_bytes > (1L << 24)) return true;
    return false;
}
static inline bool few_rows(const sarXattn* a) { return (long)a->Tq * (a->Hq / a->Hkv) <= 32; }
// key slices: as many as give every CU a block, of 256 keys at least; more (up to `blocks` blocks, which evens out ragged lengths) only of 1024 keys,
// eight tiles a wave, below which a block's start costs more than its work; 64 at most (one lane each in the joining kernel)
static inline int key_splits(const sarXattn* a, int rows_per_block, int blocks) {
    const long R = (long)a->Tq * (a->Hq / a->Hkv), tiles = (R + rows_per_block - 1) / rows_per_block * a->B * a->Hkv;
    const auto least = [](long x, long y) { return x < y ? x : y; };
    const long few = least((256 + tiles - 1) / tiles, (a->Tk + 255L) / 256), many = least((blocks + tiles - 1) / tiles, (a->Tk + 1023L) / 1024);
    const long s = few > many ? few : many;
    return (int)(s < 1 ? 1 : s > 64 ? 64 : s);
}
// a few rows: a second launch (joining slices: 5 us) costs more than going on until each of a block's `waves` has six 32-key tiles (three of fp32, whose
// products take longer), or eight where the blocks fill the chip by themselves.  8-bit, 4 x 2000, 4 heads of 64: bf16 10.4 in one slice, 9.4 in eight,
// fp32 16.2 and 10.8; bf16 64 x 1140, 8 heads: 16 and 19; fp32 keys, 1 x 450, 8 heads of 128: 39 and 25
static inline int step_splits(const sarXattn* a, int waves, bool fp32) {
    const long tiles = ((long)a->Tq * (a->Hq / a->Hkv) + 31) / 32 * a->B * a->Hkv;
    return a->Tk <= waves * (tiles >= 256 ? 256 : fp32 ? 96 : 192) ? 1 : key_splits(a, 32, 1024);
}
// the forward for many rows: four waves on 128 rows where those blocks fill the chip's 256 CUs twice; else two pairs of waves on 64; the key axis
// is cut only where even those are fewer than the CUs (partial results cost their writing and reading)
struct FwdPlan { int waves, splits; };
static inline FwdPlan fwd_plan(const sarXattn* a) {
    const long R = (long)a->Tq * (a->Hq / a->Hkv), bh = (long)a->B * a->Hkv;
    if (R > 64 && (R + 127) / 128 * bh >= 512) return {4, 1};
    return {2, (R + 63) / 64 * bh >= 192 ? 1 : key_splits(a, 64, 384)};
}
// The backward of up to SMALL_KEYS keys is one kernel (xattn.hip).  Else four waves on 128 columns where those blocks fill the chip twice, two pairs on
// 64 where not.  Where the blocks are fewer than half the CUs, the streamed axis (keys for dQ, the rows of all the group's heads for dK, dV) is cut
// into slices of two steps of 64 at least, up to a block per CU, whose fp32 sums a further launch adds: bf16 1 x 400 x 400, 4 heads of 64: 19.3 ->
// 17.6 us, fp32 64 -> 38; slices for two blocks per CU gained nothing (32 x 16 steps of 128-wide heads 42 -> 52 us).
constexpr int SUMMED_KEYS = 256, SMALL_KEYS = 64;
struct BwdPlan { bool few_q, few_k; int dq_slices, dkv_slices; size_t dq_at, dkv_at, bytes; };
static inline int cut_slices(long blocks, long steps) {
    const long want = blocks < 1 ? 1 : 256 / blocks, most = steps / 2;         // (no blocks: no keys)
    return want < 2 || most < 2 ? 1 : (int)(want < most ? want : most);
}
static inline BwdPlan bwd_plan(const sarXattn* a) {
    BwdPlan p = {};
    const long R = (long)a->Tq * (a->Hq / a->Hkv), bh = (long)a->B * a->Hkv;
    p.few_q = R <= 64 || (R + 127) / 128 * bh < 512;
    p.few_k = (a->Tk + 127) / 128 * bh < 512;
    p.dq_slices = a->Tk <= SUMMED_KEYS ? 1 : cut_slices((R + 63) / 64 * bh, (a->Tk + 63) / 64);
    p.dkv_slices = cut_slices((a->Tk + 63) / 64 * bh, (a->Tq + 63) / 64 * (long)(a->Hq / a->Hkv));
    const auto up = [](size_t n) { return (n + 255) & ~(size_t)255; };
    p.dq_at = up(8 * (size_t)a->B * a->Hq * a->Tq);
    p.dkv_at = p.dq_at + (p.dq_slices > 1 ? up(4 * (size_t)p.dq_slices * a->B * a->Tq * a->Hq * a->D) : 0);
    p.bytes = p.dkv_at + (p.dkv_slices > 1 ? 8 * (size_t)p.dkv_slices * a->B * a->Tk * a->Hkv * a->D : 0);
    return p;
}
static inline size_t part_bytes(const sarXattn* a, int splits) {
    return splits > 1 ? 4 * (size_t)part_floats((long)a->B * a->Hq * a->Tq, a->D, splits) : 0;
}
static inline bool bad_workspace(const sarXattn* a, size_t need) { return need && (!a->ws || (uintptr_t)a->ws % 16 || a->ws_bytes < 0 || (size_t)a->ws_bytes < need); }

// four consecutive values of a row
template <typename T> __device__ __forceinline__ void store4(T* p, float x, float y, float z, float w) {
    typename Num<T>::x4 v;
    v[0] = (T)x; v[1] = (T)y; v[2] = (T)z; v[3] = (T)w;
    *reinterpret_cast<typename Num<T>::x4*>(p) = v;
}

}  // namespace attn
