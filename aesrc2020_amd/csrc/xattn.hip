// Cross attention of decoder tokens to an encoder's states: forward and backward for many rows (xattn_step.hip: a few rows).
//
//   s_ij = scale q_i . k_j (j < k_len)    p = softmax_j s    o_i = sum_j p_ij v_j    lse_i = log sum_j exp s_ij
//   dv_j = sum_i p_ij do_i    dp_ij = do_i . v_j    delta_i = do_i . o_i    ds = p (dp - delta)
//   dq_i = scale sum_j ds_ij k_j    dk_j = scale sum_i ds_ij q_i
//
// One pass over the keys with the running maximum and sum (scores never leave the registers); the backward recomputes p from lse.
// Compiled once per element type: SAR_ELT 0 = fp32, 1 = bf16, 2 = fp16.
#include "xattn.h"

#if SAR_ELT == 0
typedef float elt;
#define SAR_FN(n) n##_f32
#elif SAR_ELT == 1
typedef __bf16 elt;
#define SAR_FN(n) n##_bf16
#else
typedef _Float16 elt;
#define SAR_FN(n) n##_f16
#endif

int SAR_FN(xattn_step)(const sarXattn* a, hipStream_t stream);       // xattn_step.hip
int SAR_FN(xattn_combine)(const sarXattn* a, int splits, hipStream_t stream);

namespace attn {

// Streamed tiles: rows of the streamed side per step, two buffers.  WN waves of a block hold different columns n (32 each), WM = 4 / WN waves share
// columns and take different 32-row parts of every step; their sums are added through LDS at the end.
template <typename T, int WN> constexpr int step_rows() { return sizeof(T) == 4 && WN == 4 ? 32 : 64; }
// two waves per SIMD where the accumulators and fragments leave room for it: the compiler then keeps everything in one register file
template <typename T, int DP> constexpr int min_waves() { return sizeof(T) == 4 && DP > 64 ? 1 : 2; }

template <int N> __device__ __forceinline__ void clear(f32x16 (&o)[N]) {
#pragma unroll
    for (int d = 0; d < N; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[d][i] = 0.f;
}
__device__ __forceinline__ f32x16 zero16() {
    f32x16 z;
#pragma unroll
    for (int i = 0; i < 16; ++i) z[i] = 0.f;
    return z;
}
// accumulators to and from LDS, one float per lane and place
template <int N> __device__ __forceinline__ void put(float* p, const f32x16 (&o)[N], int lane) {
#pragma unroll
    for (int d = 0; d < N; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) p[(d * 16 + i) * 64 + lane] = o[d][i];
}
template <int N> __device__ __forceinline__ void add(const float* p, f32x16 (&o)[N], int lane) {
#pragma unroll
    for (int d = 0; d < N; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[d][i] += p[(d * 16 + i) * 64 + lane];
}
// Loads that a loop uses are waited for before it: inside, the wait would be for the tiles that the loop has under way too (the compiler counts
// its own loads only).
template <int N> __device__ __forceinline__ void settle(u32x4 (&f)[N]) {
#pragma unroll
    for (int c = 0; c < N; ++c) asm volatile("" : "+v"(f[c]));
}
// The lane's number as a value the compiler knows nothing of: what depends on it (the tile reads' addresses) is computed again in every step instead of
// being held in registers, where those are short.
template <bool SHORT> __device__ __forceinline__ int again(int lane) {
    if constexpr (SHORT) asm volatile("" : "+v"(lane));
    return lane;
}
// the row tiles of a group's heads, one head after the other
struct RowTile { int g, t; };
__device__ __forceinline__ RowTile after(RowTile r, int rows, int tl) { return r.t + rows >= tl ? RowTile{r.g + 1, 0} : RowTile{r.g, r.t + rows}; }
// a wave's column of D values: lane holds column n, values 32 d + 8 i + 4 h + (0..3)
template <typename T, int ND> __device__ __forceinline__ void store_column(T* p, const f32x16 (&o)[ND], float f, bool in, int D, int h) {
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int dd = 32 * d + 8 * i + 4 * h;
            if (dd < D) store4<T>(p + dd, in ? o[d][4 * i] * f : 0.f, in ? o[d][4 * i + 1] * f : 0.f, in ? o[d][4 * i + 2] * f : 0.f, in ? o[d][4 * i + 3] * f : 0.f);
        }
}

// ---- fp16 operands of the gradients' second products.  ds of a mean over a batch (p of 1 / Tk, dout of 1e-4) is far below fp16's normal numbers, and the
// largest ds lies above the largest dq: as they are, dout of 1e-4 cost dq 1.4 % at 1140 keys, and ds past 65504 was infinite.  So p, 1 at most, is
// held times 2^15 (its exponent says so), and ds under a power of two of its column (a row for dQ, a key for dK) besides: as a softmax's maximum that
// follows the largest |ds| so far, puts it into [2^4, 2^15], and takes the sums along when it changes, which hardly a tile makes it do.
// bf16 and fp32 have the range.  It costs 16-bit training 0 to 5 % (8 x 1024 x 4096 of 128: forward and backward 1204 -> 1235 us; 4 x 300 x 2000 of 64:
// 70.5 -> 73.5), 8 % where 128-wide heads spill (8 x 1000 x 200: 97 -> 105); with the maximum kept within 2^2 of the limit twice that.
template <typename T> constexpr bool narrow() { return __is_same(T, _Float16); }
template <typename T> constexpr float p_bits() { return narrow<T>() ? 15.f : 0.f; }
template <typename T> constexpr float p_down() { return narrow<T>() ? 1.f / 32768.f : 1.f; }
constexpr float DS_MOST = 32768.f, DS_UP = 1.152921504606846976e18f;            // 2^60, above what any ds that reaches a result needs; |ds| < 2^56 of fp16 inputs
__device__ __forceinline__ float largest(const f32x16& x) {
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < 16; i += 2) top = fmaxf(fmaxf(top, fabsf(x[i])), fabsf(x[i + 1]));
    return top;
}
// the power of two that puts `top` into [2^(bits - 1), 2^bits), DS_UP at most
__device__ __forceinline__ float raise(float top, int bits) {
    int e = 0;
    (void)frexpf(top, &e);
    return top == 0.f ? DS_UP : fminf(ldexpf(1.f, bits - e), DS_UP);
}
template <typename T, int N> __device__ __forceinline__ void times(f32x16 (&o)[N], float f) {
    if constexpr (narrow<T>()) {
#pragma unroll
        for (int d = 0; d < N; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[d][i] *= f;
    }
}
// pack (attn_tiles.h) of s f (fp16; the others: of s)
template <typename T> __device__ __forceinline__ void pack_times(const f32x16& s, float f, u32x4* p) {
    if constexpr (narrow<T>()) {
        f32x16 up;
#pragma unroll
        for (int i = 0; i < 16; ++i) up[i] = s[i] * f;
        pack<T>(up, p);
    } else pack<T>(s, p);
}
template <typename T> struct ColumnScale {
    float f = narrow<T>() ? DS_UP : 1.f;
    // room for ds f, of which `top` is the largest that the lane has; the sums come along.  -> what to multiply ds f with once more
    template <int N> __device__ __forceinline__ float fit(float top, f32x16 (&sums)[N]) {
        top = half_max(top);
        const float g = top > DS_MOST ? fminf(raise(top, 5), 1.f) : 1.f;
        times<T>(sums, g);
        f *= g;
        return g;
    }
};

// ---- forward: a block takes 32 WN rows (as columns n) against one slice of the keys
template <typename T, int DP, int WN> __global__ __launch_bounds__(256, (min_waves<T, DP>())) void xattn_fwd_kernel(sarXattn a, int row_tiles, int splits) {
    constexpr int KT = step_rows<T, WN>(), P = pitch<T, DP>(), NC = DP * (int)sizeof(T) / 32, ND = DP / 32, WM = 4 / WN, NS = KT / 32 / WM, TILE = KT * P;
    __shared__ __attribute__((aligned(1024))) char lds[4 * TILE];                // K, V; two of each
    const int item = xcd_item(a.B * a.Hkv * splits * row_tiles);
    if (item < 0) return;
    const int rt = item % row_tiles, sp = item / row_tiles % splits, bh = item / row_tiles / splits;
    const int b = bh / a.Hkv, hk = bh % a.Hkv;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, h = lane >> 5, n = lane & 31, wn = w % WN, wm = w / WN;
    const int R = a.Tq * (a.Hq / a.Hkv), row0 = (rt * WN + wn) * 32, r = row0 + n;
    const int rl = live_rows(a, b), len = live_keys(a, b);
    const int per = ((len + KT - 1) / KT + splits - 1) / splits * KT;
    const int k0 = min(sp * per, len), k1 = rt * 32 * WN < rl ? min(k0 + per, len) : k0;
    const Row me = row_of(a, hk, min(r, R - 1));
    // scores by |scale|, the sign in the queries: the maximum of the products is then the maximum of the scores
    const float sl = score_factor(a);

    const unsigned ks = (unsigned)(a.k_st * sizeof(T)), vs = (unsigned)(a.v_st * sizeof(T)), db = (unsigned)(a.D * sizeof(T));
    const TileLoader<P, KT> tk(ks, db), tv(vs, db);
    const T* kb = reinterpret_cast<const T*>(a.k) + b * a.k_sb + hk * a.k_sh;
    const T* vb = reinterpret_cast<const T*>(a.v) + b * a.v_sb + hk * a.v_sh;
    const auto load = [&](int j, char* to) {
        tk.load(kb + j * a.k_st, k1 - j, ks, db, to, w);
        tv.load(vb + j * a.v_st, k1 - j, vs, db, to + TILE, w);
    };
    if (k0 < k1) load(k0, lds);
    u32x4 qf[NC];
    load_row<T, DP>(reinterpret_cast<const T*>(a.q) + b * a.q_sb + me.t * a.q_st + me.h * a.q_sh, r < rl, a.D, h, qf, a.scale < 0.f);
    f32x16 o[ND];
    clear(o);
    float m = NO_MAX, l = 0.f;
    bool large = false;
    int cur = 0;
    for (int j = k0; j < k1; j += KT, cur ^= 2 * TILE) {
        tile_barrier();
        if (j + KT < k1) load(j + KT, lds + (cur ^ (2 * TILE)));
        if (row0 >= rl || (WM > 1 && j + 32 * wm >= k1)) continue;
        const char *lk = lds + cur, *lv = lds + cur + TILE;
        f32x16 s[NS];
        float top = NO_MAX;
#pragma unroll
        for (int u = 0; u < NS; ++u) {
            s[u] = zero16();
#pragma unroll
            for (int c = 0; c < NC; ++c) s[u] = mma<T>(frag<P>(lk, 32 * (u * WM + wm) + n, c, h), qf[c], s[u]);
        }
        if (j + KT > k1) {
#pragma unroll
            for (int u = 0; u < NS; ++u)
#pragma unroll
                for (int i = 0; i < 16; ++i) s[u][i] = j + 32 * (u * WM + wm) + 8 * (i >> 2) + 4 * h + (i & 3) < k1 ? s[u][i] : -INFINITY;
        }
#pragma unroll
        for (int u = 0; u < NS; ++u)
#pragma unroll
            for (int i = 0; i < 16; ++i) top = fmaxf(top, s[u][i]);
        top = half_max(top) * sl;
        if (__any(top - m > lag<T>())) {
            const float mn = fmaxf(m, reference<T>(top)), f = __builtin_amdgcn_exp2f(m - mn);
            m = mn; l *= f;
            large = __any(fabsf(m) > LARGE && m != NO_MAX);
#pragma unroll
            for (int d = 0; d < ND; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[d][i] *= f;
        }
        exponents(s, sl, m, large);
#pragma unroll
        for (int u = 0; u < NS; ++u) {
#pragma unroll
            for (int i = 0; i < 16; ++i) { s[u][i] = __builtin_amdgcn_exp2f(s[u][i]); l += s[u][i]; }
            u32x4 p[4];
            pack<T>(s[u], p);
#pragma unroll
            for (int d = 0; d < ND; ++d) o[d] = mma_down<T, P>(lv, 32 * (u * WM + wm), d, p, o[d], lane);
        }
    }
    if constexpr (WM > 1) {                                       // two waves per column: bring both to one maximum, add
        static_assert(WM == 2, "");
        float* join = reinterpret_cast<float*>(lds) + wn * (ND * 16 + 2) * 64;
        static_assert(WN * (ND * 16 + 2) * 64 * 4 <= 4 * TILE, "");
        __syncthreads();
        if (wm) {
            put(join, o, lane);
            join[ND * 1024 + lane] = m; join[ND * 1024 + 64 + lane] = l;
        }
        __syncthreads();
        if (wm) return;
        const float m2 = join[ND * 1024 + lane], mn = fmaxf(m, m2), f = __builtin_amdgcn_exp2f(m - mn), g = __builtin_amdgcn_exp2f(m2 - mn);
        l = l * f + join[ND * 1024 + 64 + lane] * g;
        m = mn;
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[d][i] = o[d][i] * f + join[(d * 16 + i) * 64 + lane] * g;
    }
    l = half_sum(l);
    if (r >= R) return;
    if (splits == 1) {
        const bool in = r < rl && l != 0.f;                       // rows behind the length, and rows without keys: zeros
        store_column<T, ND>(reinterpret_cast<T*>(a.out) + b * a.o_sb + me.t * a.o_st + me.h * a.o_sh, o, 1.f / l, in, a.D, h);
        if (a.lse && h == 0) a.lse[stat_at(a, b, me)] = in ? m * LN2 + logf(l) : -INFINITY;
    } else {
        const long rows = (long)a.B * a.Hq * a.Tq, at = sp * rows + stat_at(a, b, me);
        store_column<float, ND>(reinterpret_cast<float*>(a.ws) + at * a.D, o, 1.f, true, a.D, h);
        float* ml = reinterpret_cast<float*>(a.ws) + splits * rows * a.D + at;
        if (h == 0) { ml[0] = m; ml[splits * rows] = l; }
    }
}

// ---- dQ (and delta): as the forward, a wave holds 32 rows as columns n, the keys and values stream through LDS.  It also leaves {lse log2 e,
// delta} of every row in `stats` (B, Hq, Tq, 2) for the dK, dV kernel.
// delta = do . o takes o as the forward rounded it, an error of half a step of |do . o| that is lost among many keys but not among few (bf16, 10
// keys: the gradients 1.7 times as far from float64 as their own rounding; now 1.4).  SUMMED: a first pass over the keys sums p dp instead, used up to
// SUMMED_KEYS keys of a 16-bit type (one slice).
template <typename T, int DP, int WN, bool SUMMED>
__global__ __launch_bounds__(256, (min_waves<T, DP>())) void xattn_dq_kernel(sarXattn a, float2* __restrict__ stats, float* __restrict__ part, int row_tiles, int slices) {
    constexpr int KT = step_rows<T, WN>(), P = pitch<T, DP>(), NC = DP * (int)sizeof(T) / 32, ND = DP / 32, WM = 4 / WN, NS = KT / 32 / WM, TILE = KT * P;
    __shared__ __attribute__((aligned(1024))) char lds[4 * TILE];
    __shared__ float joined[SUMMED ? WM : 1][WN][64];
    const int item = xcd_item(a.B * a.Hkv * slices * row_tiles);
    if (item < 0) return;
    const int rt = item % row_tiles, sp = item / row_tiles % slices, bh = item / row_tiles / slices, b = bh / a.Hkv, hk = bh % a.Hkv;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, h = lane >> 5, n = lane & 31, wn = w % WN, wm = w / WN;
    const int R = a.Tq * (a.Hq / a.Hkv), row0 = (rt * WN + wn) * 32, r = row0 + n;
    // (one key: its probability is 1 whatever the score, so nothing flows to the queries)
    const int rl = live_rows(a, b), keys = live_keys(a, b), all_keys = rt * 32 * WN < rl && keys > 1 ? keys : 0;
    const int per = ((all_keys + KT - 1) / KT + slices - 1) / slices * KT, k0 = min(sp * per, all_keys), len = min(per, all_keys - k0);      // this slice's keys
    const Row me = row_of(a, hk, min(r, R - 1));
    const float sl = a.scale * LOG2E;
    const unsigned ks = (unsigned)(a.k_st * sizeof(T)), vs = (unsigned)(a.v_st * sizeof(T)), db = (unsigned)(a.D * sizeof(T));
    const TileLoader<P, KT> tk(ks, db), tv(vs, db);
    const T* kb = reinterpret_cast<const T*>(a.k) + b * a.k_sb + hk * a.k_sh + k0 * a.k_st;
    const T* vb = reinterpret_cast<const T*>(a.v) + b * a.v_sb + hk * a.v_sh + k0 * a.v_st;
    const auto load = [&](int j, char* to) {
        tk.load(kb + j * a.k_st, len - j, ks, db, to, w);
        tv.load(vb + j * a.v_st, len - j, vs, db, to + TILE, w);
    };
    if (0 < len) load(0, lds);
    u32x4 qf[NC], gf[NC];
    float e = 0.f, dl = 0.f;
    {
        u32x4 of[NC];
        load_row<T, DP>(reinterpret_cast<const T*>(a.q) + b * a.q_sb + me.t * a.q_st + me.h * a.q_sh, r < rl, a.D, h, qf);
        load_row<T, DP>(reinterpret_cast<const T*>(a.dout) + b * a.g_sb + me.t * a.g_st + me.h * a.g_sh, r < rl, a.D, h, gf);
        load_row<T, DP>(reinterpret_cast<const T*>(a.out) + b * a.o_sb + me.t * a.o_st + me.h * a.o_sh, r < rl, a.D, h, of);
        if (r < rl) e = backward_exponent(a.lse[stat_at(a, b, me)], p_bits<T>());
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int i = 0; i < Num<T>::PER; ++i) dl = fmaf((float)as16<T>(gf[c])[i], (float)as16<T>(of[c])[i], dl);
        dl = half_sum(dl);
    }
    const bool summed = SUMMED && len > 0;
    if (!summed && sp == 0 && wm == 0 && h == 0 && r < R) stats[stat_at(a, b, me)] = make_float2(e, dl);
    f32x16 dq[ND];
    clear(dq);
    ColumnScale<T> up;
    float sum = 0.f;
    int cur = 0;
    bool first = summed;                                          // the pass that sums p dp
    for (int j = 0; j < len; cur ^= 2 * TILE) {
        const int next = SUMMED && first && j + KT >= len ? 0 : j + KT;
        tile_barrier();
        if (next < len) load(next, lds + (cur ^ (2 * TILE)));
        const int at_key = j;
        const bool summing = first;
        j = next;
        if (SUMMED && next == 0) first = false;
        if (SUMMED && summed && !summing && at_key == 0) {        // the first pass is over: delta from all keys
            sum = half_sum(sum);
            if constexpr (SUMMED && WM > 1) {
                joined[wm][wn][lane] = sum;
                __syncthreads();
                sum = joined[0][wn][lane] + joined[1][wn][lane];
            }
            dl = sum * p_down<T>();
            if (wm == 0 && h == 0 && r < R) stats[stat_at(a, b, me)] = make_float2(e, dl);
        }
        if (row0 >= rl || (WM > 1 && at_key + 32 * wm >= len)) continue;
        const char *lk = lds + cur, *lv = lds + cur + TILE;
#pragma unroll
        for (int u = 0; u < NS; ++u) {
            const int at = 32 * (u * WM + wm);
            const int lane = again<SUMMED && DP == 128>(threadIdx.x & 63), h = lane >> 5, n = lane & 31;
            f32x16 s = zero16(), dp = zero16();
#pragma unroll
            for (int c = 0; c < NC; ++c) s = mma<T>(frag<P>(lk, at + n, c, h), qf[c], s);
#pragma unroll
            for (int c = 0; c < NC; ++c) dp = mma<T>(frag<P>(lv, at + n, c, h), gf[c], dp);
            if (at_key + KT > len) {                              // (a key behind the length is a zero row: its p is no number to be trusted)
#pragma unroll
                for (int i = 0; i < 16; ++i) s[i] = at_key + at + 8 * (i >> 2) + 4 * h + (i & 3) < len ? fmaf(s[i], sl, -e) : -INFINITY;
            } else {
#pragma unroll
                for (int i = 0; i < 16; ++i) s[i] = fmaf(s[i], sl, -e);
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = __builtin_amdgcn_exp2f(s[i]);
            if (SUMMED && summing) {
#pragma unroll
                for (int i = 0; i < 16; ++i) sum = fmaf(s[i], dp[i], sum);
                continue;
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) dp[i] = s[i] * (narrow<T>() ? fmaf(dp[i], up.f, -dl * up.f) : dp[i] - dl);
            if constexpr (narrow<T>()) {
                const float top = largest(dp);
                if (__builtin_expect(__any(top > DS_MOST), 0)) {
                    const float g = up.fit(top, dq);
#pragma unroll
                    for (int i = 0; i < 16; ++i) dp[i] *= g;
                }
            }
            u32x4 df[4];
            pack<T>(dp, df);
#pragma unroll
            for (int d = 0; d < ND; ++d) dq[d] = mma_down<T, P>(lk, at, d, df, dq[d], lane);
        }
    }
    times<T>(dq, p_down<T>() / up.f);
    if constexpr (WM > 1) {
        static_assert(WM == 2, "");
        float* join = reinterpret_cast<float*>(lds) + wn * ND * 1024;
        static_assert(WN * ND * 1024 * 4 <= 4 * TILE, "");
        __syncthreads();
        if (wm) put(join, dq, lane);
        __syncthreads();
        if (wm) return;
        add(join, dq, lane);
    }
    if (r >= R) return;
    const long at = (((long)b * a.Tq + me.t) * a.Hq + me.h) * a.D;
    if (slices == 1) store_column<T, ND>(reinterpret_cast<T*>(a.dq) + at, dq, a.scale, r < rl, a.D, h);
    else store_column<float, ND>(part + sp * ((long)a.B * a.Tq * a.Hq * a.D) + at, dq, a.scale, r < rl, a.D, h);
}

// ---- dK, dV: a wave holds 32 keys as columns n; the rows of one query head after the other stream through LDS
template <typename T, int DP, int WN>
__global__ __launch_bounds__(256, (min_waves<T, DP>())) void xattn_dkv_kernel(sarXattn a, const float2* __restrict__ stats, float* __restrict__ part, int key_tiles, int slices) {
    constexpr int WM = 4 / WN, RT = 32 * WM, P = pitch<T, DP>(), NC = DP * (int)sizeof(T) / 32, ND = DP / 32, TILE = RT * P, BUF = 2 * TILE;
    __shared__ __attribute__((aligned(1024))) char lds[2 * BUF];                 // Q, dO; two of each
    __shared__ __attribute__((aligned(16))) float2 row_stats[2][RT];
    // 128 wide, both fragments and both sums do not fit 256 registers: the K fragments stay in the wave's own piece of LDS, in lane order
    constexpr bool KL = sizeof(T) == 2 && DP == 128;
    __shared__ __attribute__((aligned(16))) u32x4 k_frags[KL ? 4 : 1][KL ? NC : 1][KL ? 64 : 1];
    const int item = xcd_item(a.B * a.Hkv * slices * key_tiles);
    if (item < 0) return;
    const int kt = item % key_tiles, sp = item / key_tiles % slices, bh = item / key_tiles / slices, b = bh / a.Hkv, hk = bh % a.Hkv, G = a.Hq / a.Hkv;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, h = lane >> 5, n = lane & 31, wn = w % WN, wm = w / WN;
    const int len = live_keys(a, b), key0 = (kt * WN + wn) * 32, key = key0 + n;
    const int tl = kt * 32 * WN < len ? live_rows(a, b) / G : 0;                 // tokens
    // the row tiles of all heads, one after the other, cut into slices
    const int across = (tl + RT - 1) / RT, tiles = across * G, per = (tiles + slices - 1) / slices, i0 = min(sp * per, tiles), i1 = min(i0 + per, tiles);
    const float sl = a.scale * LOG2E;
    const unsigned qs = (unsigned)(a.q_st * sizeof(T)), gs = (unsigned)(a.g_st * sizeof(T)), db = (unsigned)(a.D * sizeof(T));
    const TileLoader<P, RT> tq(qs, db), tg(gs, db);
    const T* qb = reinterpret_cast<const T*>(a.q) + b * a.q_sb + (long)hk * G * a.q_sh;
    const T* gb = reinterpret_cast<const T*>(a.dout) + b * a.g_sb + (long)hk * G * a.g_sh;
    const float2* sb = stats + ((long)b * a.Hq + hk * G) * a.Tq;
    const auto load = [&](RowTile r, char* to) {
        tq.load(qb + r.g * a.q_sh + r.t * a.q_st, tl - r.t, qs, db, to, w);
        tg.load(gb + r.g * a.g_sh + r.t * a.g_st, tl - r.t, gs, db, to + TILE, w);
    };
    // {lse log2 e, delta} of the tile's rows.  Rows behind the last one get zeros as their Q and dO do: p = exp2(0), which meets zero rows.
    const auto load_stats = [&](RowTile r) {
        return sb[(long)r.g * a.Tq + min(r.t + (int)threadIdx.x % RT, tl - 1)];
    };
    // one key: p = 1 whatever the score (s 0 - 0, or times 2^p_bits), and ds = 0 (dK is stored as zero)
    const float sk = len == 1 ? 0.f : sl;
    const auto put_stats = [&](int to, RowTile r, float2 v) {
        const bool in = r.t + (int)threadIdx.x < tl;
        if (threadIdx.x < RT) row_stats[to][threadIdx.x] = make_float2(in && len > 1 ? v.x : -p_bits<T>(), in ? v.y : 0.f);
    };
    // (statistics are fetched two steps ahead and put right behind a barrier, where nothing has to be waited for)
    RowTile at_row = {0, 0}, next_row = {0, 0};
    float2 next = make_float2(0.f, 0.f);
    if (i0 < i1) {
        at_row = {i0 / across, (i0 - i0 / across * across) * RT};
        next_row = after(at_row, RT, tl);
        load(at_row, lds);
        put_stats(0, at_row, load_stats(at_row));
        next = load_stats(i0 + 1 < i1 ? next_row : at_row);
    }
    u32x4 kf[NC], vf[NC];
    load_row<T, DP>(reinterpret_cast<const T*>(a.k) + b * a.k_sb + min(key, a.Tk - 1) * a.k_st + hk * a.k_sh, key < len, a.D, h, kf);
    if constexpr (KL) {
#pragma unroll
        for (int c = 0; c < NC; ++c) k_frags[w][c][lane] = kf[c];
    }
    load_row<T, DP>(reinterpret_cast<const T*>(a.v) + b * a.v_sb + min(key, a.Tk - 1) * a.v_st + hk * a.v_sh, key < len, a.D, h, vf);
    if constexpr (!KL) settle(kf);
    settle(vf);
    f32x16 dk[ND], dv[ND];
    clear(dk); clear(dv);
    ColumnScale<T> up;
    int cur = 0, par = 0;
    for (int i = i0; i < i1; ++i) {
        tile_barrier();
        const int t = at_row.t;
        at_row = next_row;
        if (i + 1 < i1) {
            put_stats(par ^ 1, at_row, next);
            load(at_row, lds + (cur ^ BUF));
            next_row = after(at_row, RT, tl);
            next = load_stats(i + 2 < i1 ? next_row : at_row);
        }
        if (key0 < len && (WM == 1 || t + 32 * wm < tl)) {
            const char *lq = lds + cur, *lg = lds + cur + TILE;
            const float* st = reinterpret_cast<const float*>(row_stats[par]) + wm * 64;
            f32x16 s = zero16(), dp = zero16();
#pragma unroll
            for (int c = 0; c < NC; ++c) s = mma<T>(frag<P>(lq, 32 * wm + n, c, h), KL ? k_frags[w][KL ? c : 0][KL ? lane : 0] : kf[c], s);
#pragma unroll
            for (int x = 0; x < 4; ++x)
#pragma unroll
                for (int c = 0; c < 4; ++c) s[4 * x + c] = fmaf(s[4 * x + c], sk, -st[2 * (8 * x + 4 * h + c)]);
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = __builtin_amdgcn_exp2f(s[i]);
            u32x4 pf[4];
            pack<T>(s, pf);
#pragma unroll
            for (int d = 0; d < ND; ++d) dv[d] = mma_down<T, P>(lg, 32 * wm, d, pf, dv[d], lane);
#pragma unroll
            for (int c = 0; c < NC; ++c) dp = mma<T>(frag<P>(lg, 32 * wm + n, c, h), vf[c], dp);
#pragma unroll
            for (int x = 0; x < 4; ++x)
#pragma unroll
                for (int c = 0; c < 4; ++c) dp[4 * x + c] = s[4 * x + c] * (dp[4 * x + c] - st[2 * (8 * x + 4 * h + c) + 1]);
            if constexpr (narrow<T>()) {
                const float top = key < len ? largest(dp) * up.f : 0.f;
                if (__builtin_expect(__any(top > DS_MOST), 0)) up.fit(top, dk);
            }
            pack_times<T>(dp, up.f, pf);
#pragma unroll
            for (int d = 0; d < ND; ++d) dk[d] = mma_down<T, P>(lq, 32 * wm, d, pf, dk[d], lane);
        }
        cur ^= BUF; par ^= 1;
    }
    times<T>(dk, p_down<T>() / up.f);
    times<T>(dv, p_down<T>());
    if constexpr (WM > 1) {
        static_assert(WM == 2, "");
        float* join = reinterpret_cast<float*>(lds) + wn * 2 * ND * 1024;
        static_assert(WN * 2 * ND * 1024 * 4 <= 2 * BUF, "");
        __syncthreads();
        if (wm) { put(join, dk, lane); put(join + ND * 1024, dv, lane); }
        __syncthreads();
        if (wm) return;
        add(join, dk, lane); add(join + ND * 1024, dv, lane);
    }
    if (key >= a.Tk) return;
    const long at = (((long)b * a.Tk + key) * a.Hkv + hk) * a.D;  // frames behind the length: their gradient is zero
    if (slices == 1) {
        store_column<T, ND>(reinterpret_cast<T*>(a.dk) + at, dk, a.scale, key < len && len > 1, a.D, h);
        store_column<T, ND>(reinterpret_cast<T*>(a.dv) + at, dv, 1.f, key < len, a.D, h);
    } else {
        const long n = (long)a.B * a.Tk * a.Hkv * a.D;
        store_column<float, ND>(part + sp * n + at, dk, a.scale, key < len && len > 1, a.D, h);
        store_column<float, ND>(part + (slices + sp) * n + at, dv, 1.f, key < len, a.D, h);
    }
}

// ---- dQ, dK, dV in one launch where 64 keys are all there are: a block holds a key head's keys as two pairs of waves' columns (as above), so S and dP
// are computed once for all three gradients, and ds, through LDS, meets the keys again for dQ.  Five products a tile instead of seven, one launch
// instead of two: what fp32 (whose matrix instructions bound it) and small calls (which latency does) both need.  64 x 72 x 39, 8 heads of 64: fp32 45 ->
// 34 us, bf16 18 -> 14; 2 x 20 x 39, 4 heads, bf16: 11 -> 7; 8 x 1000 x 64, 8 heads of 128, bf16: 54 -> 43.
// delta is the sum of p dp over the keys (see xattn_dq_kernel).
template <typename T, int DP> struct Small {
    static constexpr int P = pitch<T, DP>(), TILE = 64 * P, BUFS = P <= 128 ? 2 : 1;             // (two blocks a CU in either case)
    static constexpr int DS_PITCH = 68, DS_AT = TILE + BUFS * 2 * TILE, LDS = DS_AT + 64 * DS_PITCH * 4;
};
// sums of 2 N values over the 32 lanes of a half, the values shared out on the way: lane n ends with value (n & 1) 8 + (n & 2) 2 + (n & 4) / 2 + (n & 8) / 8
template <int N> __device__ __forceinline__ float shared_sums(const float (&x)[2 * N], int lane) {
    float y[N];
    const bool up = lane & (8 / N);
#pragma unroll
    for (int i = 0; i < N; ++i) y[i] = (up ? x[i + N] : x[i]) + __shfl_xor(up ? x[i] : x[i + N], 8 / N, 64);
    if constexpr (N > 1) return shared_sums<N / 2>(y, lane);
    else return y[0] + __shfl_xor(y[0], 16, 64);
}
template <typename T, int DP> __global__ __launch_bounds__(256, 2) void xattn_small_bwd_kernel(sarXattn a, float* __restrict__ part, int slices) {
    typedef Small<T, DP> S;
    constexpr int P = S::P, NC = DP * (int)sizeof(T) / 32, ND = DP / 32, TILE = S::TILE, RT = 64, BUFS = S::BUFS;
    constexpr bool KL = P == 256;       // KL: the K fragments are read from the tile (they do not fit the registers as well)
    extern __shared__ __attribute__((aligned(1024))) char lds[];                                 // K; Q, dO (BUFS of each); ds (keys, rows) fp32
    __shared__ __attribute__((aligned(16))) float exponent[2][RT];
    __shared__ __attribute__((aligned(16))) float sums[2][RT];
    const int item = xcd_item(a.B * a.Hkv * slices);
    if (item < 0) return;
    const int sp = item % slices, bh = item / slices, b = bh / a.Hkv, hk = bh % a.Hkv, G = a.Hq / a.Hkv;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, h = lane >> 5, n = lane & 31, wn = w & 1, wm = w >> 1;
    const int len = live_keys(a, b), key0 = wn * 32, key = key0 + n;
    const int tl = len ? live_rows(a, b) / G : 0;
    const int across = (tl + RT - 1) / RT, tiles = across * G, per = (tiles + slices - 1) / slices, i0 = min(sp * per, tiles), i1 = min(i0 + per, tiles);
    const unsigned ks = (unsigned)(a.k_st * sizeof(T)), qs = (unsigned)(a.q_st * sizeof(T)), gs = (unsigned)(a.g_st * sizeof(T)), db = (unsigned)(a.D * sizeof(T));
    const T* qb = reinterpret_cast<const T*>(a.q) + b * a.q_sb + (long)hk * G * a.q_sh;
    const T* gb = reinterpret_cast<const T*>(a.dout) + b * a.g_sb + (long)hk * G * a.g_sh;
    const float* lse = a.lse + ((long)b * a.Hq + hk * G) * a.Tq;
    const T* kb = reinterpret_cast<const T*>(a.k) + b * a.k_sb + hk * a.k_sh;
    const TileLoader<P, RT> tq(qs, db), tg(gs, db);
    const auto load = [&](RowTile r, char* to) {
        tq.load(qb + r.g * a.q_sh + r.t * a.q_st, tl - r.t, qs, db, to, w);
        tg.load(gb + r.g * a.g_sh + r.t * a.g_st, tl - r.t, gs, db, to + TILE, w);
    };
    // lse log2 e of the tile's rows.  One key: p = 1 whatever the score, and ds = 0 (dQ, dK are stored as zero).
    // A key behind the length is a zero row: its p, which dQ and delta would meet, is made 0.
    const float sk = len == 1 ? 0.f : a.scale * LOG2E, none = key < len ? 0.f : -INFINITY;
    const auto load_lse = [&](RowTile r) {
        return lse[(long)r.g * a.Tq + min(r.t + (int)threadIdx.x % RT, tl - 1)];
    };
    const auto put_lse = [&](int to, RowTile r, float v) {
        if (threadIdx.x < RT) exponent[to][threadIdx.x] = len > 1 && r.t + (int)threadIdx.x < tl ? backward_exponent(v, p_bits<T>()) : -p_bits<T>();
    };
    char* const tiles_at = lds + TILE;
    float* const ds_at = reinterpret_cast<float*>(lds + S::DS_AT);
    RowTile at_row = {0, 0}, next_row = {0, 0};
    float next = 0.f;
    if (i0 < i1) {
        at_row = {i0 / across, (i0 - i0 / across * across) * RT};
        next_row = after(at_row, RT, tl);
        TileLoader<P, RT>(ks, db).load(kb, len, ks, db, lds, w);
        load(at_row, tiles_at);
        put_lse(0, at_row, load_lse(at_row));
        next = load_lse(i0 + 1 < i1 ? next_row : at_row);
    }
    u32x4 kf[NC], vf[NC];
    if constexpr (!KL) load_row<T, DP>(kb + min(key, a.Tk - 1) * a.k_st, key < len, a.D, h, kf);
    load_row<T, DP>(reinterpret_cast<const T*>(a.v) + b * a.v_sb + min(key, a.Tk - 1) * a.v_st + hk * a.v_sh, key < len, a.D, h, vf);
    if constexpr (!KL) settle(kf);
    settle(vf);
    f32x16 dk[ND], dv[ND];
    clear(dk); clear(dv);
    ColumnScale<T> up;
    int cur = 0, par = 0;
    for (int i = i0; i < i1; ++i) {
        tile_barrier();
        const int t = at_row.t, g = at_row.g;
        at_row = next_row;
        if (i + 1 < i1) {
            put_lse(par ^ 1, at_row, next);
            if constexpr (BUFS == 2) load(at_row, tiles_at + (cur ^ (2 * TILE)));
            next_row = after(at_row, RT, tl);
            next = load_lse(i + 2 < i1 ? next_row : at_row);
        }
        const int lane = again<sizeof(T) == 2 && DP == 128>(threadIdx.x & 63), h = lane >> 5, n = lane & 31, key = key0 + n;
        const bool live = key0 < len && t + 32 * wm < tl;
        const char *lq = tiles_at + cur, *lg = tiles_at + cur + TILE;
        const float* ex = exponent[par] + 32 * wm;
        f32x16 s = zero16(), dp = zero16();
        if (live) {
#pragma unroll
            for (int c = 0; c < NC; ++c) s = mma<T>(frag<P>(lq, 32 * wm + n, c, h), KL ? frag<P>(lds, key, c, h) : kf[c], s);
#pragma unroll
            for (int x = 0; x < 4; ++x)
#pragma unroll
                for (int c = 0; c < 4; ++c) s[4 * x + c] = __builtin_amdgcn_exp2f(fmaf(s[4 * x + c], sk, none - ex[8 * x + 4 * h + c]));
            u32x4 pf[4];
            pack<T>(s, pf);
#pragma unroll
            for (int d = 0; d < ND; ++d) dv[d] = mma_down<T, P>(lg, 32 * wm, d, pf, dv[d], lane);
#pragma unroll
            for (int c = 0; c < NC; ++c) dp = mma<T>(frag<P>(lg, 32 * wm + n, c, h), vf[c], dp);
        }
        float pdp[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) pdp[i] = s[i] * dp[i];       // (a wave without keys: 0)
        const float sum = shared_sums<8>(pdp, lane);
        const int place = (lane & 1) * 8 + (lane & 2) * 2 + (lane & 4) / 2 + (lane & 8) / 8;
        if (n < 16) sums[wn][32 * wm + 8 * (place >> 2) + 4 * h + (place & 3)] = sum;
        lds_barrier();
        if (live) {
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                f32x4 v;
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const int row = 8 * x + 4 * h + c;
                    const float dl = (sums[0][32 * wm + row] + sums[1][32 * wm + row]) * p_down<T>();
                    v[c] = dp[4 * x + c] = s[4 * x + c] * (dp[4 * x + c] - dl);
                }
                *reinterpret_cast<f32x4*>(ds_at + key * S::DS_PITCH + 32 * wm + 8 * x + 4 * h) = v;
            }
            if constexpr (narrow<T>()) {
                const float top = key < len ? largest(dp) * up.f : 0.f;
                if (__builtin_expect(__any(top > DS_MOST), 0)) up.fit(top, dk);
            }
            u32x4 pf[4];
            pack_times<T>(dp, up.f, pf);
#pragma unroll
            for (int d = 0; d < ND; ++d) dk[d] = mma_down<T, P>(lq, 32 * wm, d, pf, dk[d], lane);
        }
        lds_barrier();                                            // ds is there; the reads of Q and dO are done
        if constexpr (BUFS == 1) {
            if (i + 1 < i1) load(at_row, tiles_at);
        }
        // dQ of the wave's 32 rows, every second 32 of the width
        if (t + 32 * wm < tl) {
            const int row = t + 32 * wm + n;
            T* to = reinterpret_cast<T*>(a.dq) + (((long)b * a.Tq + row) * a.Hq + hk * G + g) * a.D;
            u32x4 df[2][4];
            const auto ds_of = [&](int k, int i) { return ds_at[(32 * k + 8 * (i >> 2) + 4 * h + (i & 3)) * S::DS_PITCH + 32 * wm + n]; };
            float f = 1.f;
            if constexpr (narrow<T>()) {                          // all keys are here: the row's scale is known.  (Read twice: the registers are short.)
                float top = 0.f;
#pragma unroll
                for (int k = 0; k < 2; ++k)
                    if (32 * k < len) {
#pragma unroll
                        for (int i = 0; i < 16; ++i) top = fmaxf(top, fabsf(ds_of(k, i)));
                    }
                f = raise(half_max(top), 14);
            }
#pragma unroll
            for (int k = 0; k < 2; ++k)
                if (32 * k < len) {
                    f32x16 x;
#pragma unroll
                    for (int i = 0; i < 16; ++i) x[i] = ds_of(k, i);
                    pack_times<T>(x, f, df[k]);
                }
            const float back = a.scale * (p_down<T>() / f);
#pragma unroll
            for (int d = 0; d < ND; ++d) {
                if ((d & 1) != wn) continue;
                f32x16 q = zero16();
#pragma unroll
                for (int k = 0; k < 2; ++k)
                    if (32 * k < len) q = mma_down<T, P>(lds, 32 * k, d, df[k], q, lane);
                if (row < tl) {
                    const bool in = len > 1;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int dd = 32 * d + 8 * i + 4 * h;
                        if (dd < a.D) store4<T>(to + dd, in ? q[4 * i] * back : 0.f, in ? q[4 * i + 1] * back : 0.f, in ? q[4 * i + 2] * back : 0.f, in ? q[4 * i + 3] * back : 0.f);
                    }
                }
            }
        }
        par ^= 1;
        if (BUFS == 2) cur ^= 2 * TILE;
    }
    if (sp == 0) {                                                // rows behind the length: zeros
        const int wide = G * a.D / 4;
        for (long i = threadIdx.x; i < (long)(a.Tq - tl) * wide; i += 256) {
            const long row = i / wide;
            store4<T>(reinterpret_cast<T*>(a.dq) + (((long)b * a.Tq + tl + row) * a.Hq + hk * G) * a.D + (i - row * wide) * 4, 0.f, 0.f, 0.f, 0.f);
        }
    }
    times<T>(dk, p_down<T>() / up.f);
    times<T>(dv, p_down<T>());
    float* join = reinterpret_cast<float*>(lds) + wn * 2 * ND * 1024;
    static_assert(2 * 2 * ND * 1024 * 4 <= S::LDS, "");
    __syncthreads();
    if (wm) { put(join, dk, lane); put(join + ND * 1024, dv, lane); }
    __syncthreads();
    if (wm) return;
    add(join, dk, lane); add(join + ND * 1024, dv, lane);
    if (key >= a.Tk) return;
    const long at = (((long)b * a.Tk + key) * a.Hkv + hk) * a.D;
    if (slices == 1) {
        store_column<T, ND>(reinterpret_cast<T*>(a.dk) + at, dk, a.scale, key < len && len > 1, a.D, h);
        store_column<T, ND>(reinterpret_cast<T*>(a.dv) + at, dv, 1.f, key < len, a.D, h);
    } else {
        const long n = (long)a.B * a.Tk * a.Hkv * a.D;
        store_column<float, ND>(part + sp * n + at, dk, a.scale, key < len && len > 1, a.D, h);
        store_column<float, ND>(part + (slices + sp) * n + at, dv, 1.f, key < len, a.D, h);
    }
}

// the sliced gradients: out = sum over the slices, in their order
struct SumJob { const float* part; void* out; long n; int slices; };
struct SumJobs { SumJob j[3]; };
template <typename T> __global__ __launch_bounds__(256) void xattn_sum_kernel(SumJobs jobs) {
    const SumJob j = jobs.j[blockIdx.y];
    for (long i = ((long)blockIdx.x * 256 + threadIdx.x) * 4; i < j.n; i += (long)gridDim.x * 1024) {
        f32x4 v = {0, 0, 0, 0};
#pragma unroll 4
        for (int s = 0; s < j.slices; ++s) v += *reinterpret_cast<const f32x4*>(j.part + s * j.n + i);
        store4<T>(reinterpret_cast<T*>(j.out) + i, v[0], v[1], v[2], v[3]);
    }
}

}  // namespace attn
using namespace attn;

static bool bad(const sarXattn* a) {
    if (bad_shape(a) || bad_strides(sizeof(elt), &a->q_sb, 12) || wide_rows(sizeof(elt), {a->q_st, a->k_st, a->v_st})) return true;
    for (const void* p : {a->q, a->k, a->v, (const void*)a->out})
        if (!p || (uintptr_t)p % 16) return true;
    return false;
}

// fp32 heads wider than 64 have no two-waves-per-column form: its tiles would pass 64 KB of LDS
template <int DP> constexpr bool paired() { return sizeof(elt) == 2 || DP <= 64; }
template <int DP> static void launch_fwd(const sarXattn& a, hipStream_t st) {
    const FwdPlan p = fwd_plan(&a);
    const bool two = paired<DP>() && p.waves == 2;
    const int rt = cdiv((long)a.Tq * (a.Hq / a.Hkv), two ? 64 : 128);
    const dim3 grid((unsigned)xcd_grid((long)rt * p.splits * a.B * a.Hkv));
    if constexpr (paired<DP>()) {
        if (two) hipLaunchKernelGGL((xattn_fwd_kernel<elt, DP, 2>), grid, dim3(256), 0, st, a, rt, p.splits);
    }
    if (!two) hipLaunchKernelGGL((xattn_fwd_kernel<elt, DP, 4>), grid, dim3(256), 0, st, a, rt, p.splits);
}
template <int DP> static int launch_bwd(const sarXattn& a, hipStream_t st) {
    const BwdPlan p = bwd_plan(&a);
    const long bh = (long)a.B * a.Hkv, nq = (long)a.B * a.Tq * a.Hq * a.D, nk = (long)a.B * a.Tk * a.Hkv * a.D;
    float2* stats = reinterpret_cast<float2*>(a.ws);
    float* pq = reinterpret_cast<float*>(reinterpret_cast<char*>(a.ws) + p.dq_at);
    float* pk = reinterpret_cast<float*>(reinterpret_cast<char*>(a.ws) + p.dkv_at);
    const bool few_q = paired<DP>() && p.few_q, few_k = paired<DP>() && p.few_k;
    const int rt = cdiv((long)a.Tq * (a.Hq / a.Hkv), few_q ? 64 : 128), kt = cdiv(a.Tk, few_k ? 64 : 128);
    const dim3 gq((unsigned)xcd_grid(rt * bh * p.dq_slices)), gk((unsigned)xcd_grid(kt * bh * p.dkv_slices));
    const bool small = paired<DP>() && a.Tk > 0 && a.Tk <= SMALL_KEYS, summed = sizeof(elt) == 2 && a.Tk <= SUMMED_KEYS;
    if constexpr (paired<DP>()) {
        if (small) {
            typedef Small<elt, DP> S;
            static PerDeviceFlag raised;
            if (S::LDS > 60 * 1024 && !raised) {
                if (hipFuncSetAttribute(reinterpret_cast<const void*>(&xattn_small_bwd_kernel<elt, DP>), hipFuncAttributeMaxDynamicSharedMemorySize, S::LDS) != hipSuccess) return SAR_ELAUNCH;
                raised = true;
            }
            hipLaunchKernelGGL((xattn_small_bwd_kernel<elt, DP>), dim3((unsigned)xcd_grid(bh * p.dkv_slices)), dim3(256), S::LDS, st, a, pk, p.dkv_slices);
        }
        if (!small && few_q && !summed) hipLaunchKernelGGL((xattn_dq_kernel<elt, DP, 2, false>), gq, dim3(256), 0, st, a, stats, pq, rt, p.dq_slices);
    }
    if (!small && !few_q && !summed) hipLaunchKernelGGL((xattn_dq_kernel<elt, DP, 4, false>), gq, dim3(256), 0, st, a, stats, pq, rt, p.dq_slices);
    if constexpr (sizeof(elt) == 2) {
        if (!small && few_q && summed) hipLaunchKernelGGL((xattn_dq_kernel<elt, DP, 2, true>), gq, dim3(256), 0, st, a, stats, pq, rt, p.dq_slices);
        if (!small && !few_q && summed) hipLaunchKernelGGL((xattn_dq_kernel<elt, DP, 4, true>), gq, dim3(256), 0, st, a, stats, pq, rt, p.dq_slices);
    }
    if (kt && !small) {
        if constexpr (paired<DP>()) {
            if (few_k) hipLaunchKernelGGL((xattn_dkv_kernel<elt, DP, 2>), gk, dim3(256), 0, st, a, stats, pk, kt, p.dkv_slices);
        }
        if (!few_k) hipLaunchKernelGGL((xattn_dkv_kernel<elt, DP, 4>), gk, dim3(256), 0, st, a, stats, pk, kt, p.dkv_slices);
    }
    SumJobs sums = {};
    int n = 0;
    long most = 0;
    const auto sum = [&](const float* part, void* out, long count, int slices) {
        sums.j[n++] = {part, out, count, slices};
        most = count > most ? count : most;
    };
    if (p.dq_slices > 1) sum(pq, a.dq, nq, p.dq_slices);
    if (kt && p.dkv_slices > 1) { sum(pk, a.dk, nk, p.dkv_slices); sum(pk + p.dkv_slices * nk, a.dv, nk, p.dkv_slices); }
    if (n) hipLaunchKernelGGL((xattn_sum_kernel<elt>), dim3((unsigned)(most < 2048 * 1024 ? cdiv(most, 1024) : 2048), n), dim3(256), 0, st, sums);
    SAR_CHECK_LAUNCH();
    return SAR_OK;
}

#if SAR_ELT == 0      // the same for every type
extern "C" size_t sar_xattn_fwd_workspace_bytes(const sarXattn* a) {
    if (bad_shape(a)) return 0;
    if (!few_rows(a)) return part_bytes(a, fwd_plan(a).splits);
    const bool wide = a->elt_bytes != 2;
    const int waves = wide ? (a->D <= 32 ? 8 : a->D <= 64 ? 4 : 2) : a->D <= 64 ? 8 : 4;         // most_waves(); fp32 has the fewest
    return part_bytes(a, step_splits(a, waves, wide));
}
extern "C" size_t sar_xattn_bwd_workspace_bytes(const sarXattn* a) { return bad_shape(a) ? 0 : bwd_plan(a).bytes; }
#endif

extern "C" int SAR_FN(sar_xattn_fwd)(const sarXattn* a, hipStream_t stream) {
    if (bad(a)) return SAR_EINVAL;
    if (few_rows(a)) return SAR_FN(xattn_step)(a, stream);
    const int splits = fwd_plan(a).splits;
    if (bad_workspace(a, part_bytes(a, splits))) return SAR_EINVAL;
    if (a->D <= 32) launch_fwd<32>(*a, stream);
    else if (a->D <= 64) launch_fwd<64>(*a, stream);
    else if (a->D <= 96) launch_fwd<96>(*a, stream);
    else launch_fwd<128>(*a, stream);
    SAR_CHECK_LAUNCH();
    return splits > 1 ? SAR_FN(xattn_combine)(a, splits, stream) : SAR_OK;
}

extern "C" int SAR_FN(sar_xattn_bwd)(const sarXattn* a, hipStream_t stream) {
    if (bad(a) || !a->lse || !a->dout || !a->dq || !a->dk || !a->dv || !a->ws) return SAR_EINVAL;
    for (const void* p : {a->dout, (const void*)a->dq, (const void*)a->dk, (const void*)a->dv})
        if ((uintptr_t)p % 16) return SAR_EINVAL;
    if (bad_strides(sizeof(elt), &a->g_sb, 3) || wide_rows(sizeof(elt), {a->g_st}) || bad_workspace(a, bwd_plan(a).bytes)) return SAR_EINVAL;
    return a->D <= 32 ? launch_bwd<32>(*a, stream) : a->D <= 64 ? launch_bwd<64>(*a, stream) : a->D <= 96 ? launch_bwd<96>(*a, stream) : launch_bwd<128>(*a, stream);
}
