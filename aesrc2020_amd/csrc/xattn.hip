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

int SAR_FN(xattn_step)(const sarXattn* a, int splits, hipStream_t stream);       // xattn_step.hip
int SAR_FN(xattn_combine)(const sarXattn* a, int splits, hipStream_t stream);

namespace attn {

template <typename T> constexpr int key_tile() { return sizeof(T) == 4 ? 32 : 64; }

// rows [first, first + ROWS) of a (T, D) operand, zero from `live` on and past D, through registers into a swizzled LDS tile
template <typename T, int DP, int ROWS> struct Stage {
    static constexpr int CH = DP * (int)sizeof(T) / 16, ALL = ROWS * CH, N = (ALL + 255) / 256, P = pitch<T, DP>();
    u32x4 r[N];
    // element offset of row `row`: a plain stride, or the folded rows of the queries
    template <typename F> __device__ __forceinline__ void load(const T* base, F offset, int first, int live, int D) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int idx = threadIdx.x + 256 * i, row = first + idx / CH, ch = idx % CH;
            r[i] = u32x4{0, 0, 0, 0};
            if (row < live && ch * Num<T>::PER < D && (ALL % 256 == 0 || idx < ALL)) r[i] = *reinterpret_cast<const u32x4*>(base + offset(row) + ch * Num<T>::PER);
        }
    }
    __device__ __forceinline__ void store(char* tile) const {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int idx = threadIdx.x + 256 * i;
            if (ALL % 256 == 0 || idx < ALL) *reinterpret_cast<u32x4*>(tile + chunk_at<P>(idx / CH, idx % CH)) = r[i];
        }
    }
};

// ---- forward: a block of four waves takes 128 rows (32 a wave, as columns n) against one slice of the keys
template <typename T, int DP> __global__ __launch_bounds__(256) void xattn_fwd_kernel(sarXattn a, int row_tiles, int splits) {
    constexpr int KT = key_tile<T>(), P = pitch<T, DP>(), NC = DP * (int)sizeof(T) / 32, ND = DP / 32, NS = KT / 32;
    __shared__ __attribute__((aligned(16))) char lk[KT * P];
    __shared__ __attribute__((aligned(16))) char lv[KT * P];
    const long item = xcd_item((long)a.B * a.Hkv * splits * row_tiles);
    if (item < 0) return;
    const int rt = (int)(item % row_tiles), sp = (int)((item / row_tiles) % splits), bh = (int)(item / row_tiles / splits);
    const int b = bh / a.Hkv, hk = bh % a.Hkv;
    const int lane = threadIdx.x & 63, h = lane >> 5, n = lane & 31;
    const int R = a.Tq * (a.Hq / a.Hkv), row0 = rt * 128 + (threadIdx.x >> 6) * 32, r = row0 + n;
    const int rl = live_rows(a, b), len = live_keys(a, b);
    const int per = ((len + KT - 1) / KT + splits - 1) / splits * KT;
    const int k0 = min(sp * per, len), k1 = rt * 128 < rl ? min(k0 + per, len) : k0;
    const Row me = row_of(a, hk, min(r, R - 1));
    const float sl = a.scale * LOG2E;

    u32x4 qf[NC];
    load_row<T, DP>(reinterpret_cast<const T*>(a.q) + b * a.q_sb + me.t * a.q_st + me.h * a.q_sh, r < rl, a.D, h, qf);
    const T* kb = reinterpret_cast<const T*>(a.k) + b * a.k_sb + hk * a.k_sh;
    const T* vb = reinterpret_cast<const T*>(a.v) + b * a.v_sb + hk * a.v_sh;
    const auto krow = [&](int j) { return j * a.k_st; };
    const auto vrow = [&](int j) { return j * a.v_st; };

    f32x16 o[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[d][i] = 0.f;
    float m = NO_MAX, l = 0.f;

    Stage<T, DP, KT> sk, sv;
    sk.load(kb, krow, k0, k1, a.D); sv.load(vb, vrow, k0, k1, a.D);
    for (int j = k0; j < k1; j += KT) {
        __syncthreads();
        sk.store(lk); sv.store(lv);
        __syncthreads();
        if (j + KT < k1) { sk.load(kb, krow, j + KT, k1, a.D); sv.load(vb, vrow, j + KT, k1, a.D); }
        if (row0 >= rl) continue;
        f32x16 s[NS];
        float top = NO_MAX;
#pragma unroll
        for (int u = 0; u < NS; ++u) {
#pragma unroll
            for (int i = 0; i < 16; ++i) s[u][i] = 0.f;
#pragma unroll
            for (int c = 0; c < NC; ++c) s[u] = mma<T>(frag<P>(lk, 32 * u + n, c, h), qf[c], s[u]);
        }
        if (j + KT > k1) {
#pragma unroll
            for (int u = 0; u < NS; ++u)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const bool in = j + 32 * u + 8 * (i >> 2) + 4 * h + (i & 3) < k1;
                    s[u][i] = in ? s[u][i] * sl : -INFINITY;
                    top = fmaxf(top, s[u][i]);
                }
        } else {
#pragma unroll
            for (int u = 0; u < NS; ++u)
#pragma unroll
                for (int i = 0; i < 16; ++i) { s[u][i] *= sl; top = fmaxf(top, s[u][i]); }
        }
        top = half_max(top);
        // the maximum follows only where it grew by more than 2^8: below that p <= 2^8 loses nothing in any of the types, and most
        // tiles skip the rescaling
        if (__any(top > m + 8.f)) {
            const float mn = fmaxf(m, top), f = __builtin_amdgcn_exp2f(m - mn);
            m = mn; l *= f;
#pragma unroll
            for (int d = 0; d < ND; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[d][i] *= f;
        }
#pragma unroll
        for (int u = 0; u < NS; ++u) {
#pragma unroll
            for (int i = 0; i < 16; ++i) { s[u][i] = __builtin_amdgcn_exp2f(s[u][i] - m); l += s[u][i]; }
            u32x4 p[4];
            pack<T>(s[u], p);
#pragma unroll
            for (int d = 0; d < ND; ++d) o[d] = mma_down<T, P>(lv, 32 * u, d, p, o[d], lane);
        }
    }
    l = half_sum(l);
    if (r >= R) return;
    if (splits == 1) {
        const bool in = r < rl && l != 0.f;                       // rows behind the length, and rows without keys: zeros
        const float inv = 1.f / l;
        T* op = reinterpret_cast<T*>(a.out) + b * a.o_sb + me.t * a.o_st + me.h * a.o_sh;
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int dd = 32 * d + 8 * i + 4 * h;
                if (dd < a.D)
                    store4<T>(op + dd, in ? o[d][4 * i] * inv : 0.f, in ? o[d][4 * i + 1] * inv : 0.f, in ? o[d][4 * i + 2] * inv : 0.f, in ? o[d][4 * i + 3] * inv : 0.f);
            }
        if (a.lse && h == 0) a.lse[stat_at(a, b, me)] = in ? m * LN2 + logf(l) : -INFINITY;
    } else {
        const long rows = (long)a.B * a.Hq * a.Tq, at = sp * rows + stat_at(a, b, me);
        float* op = reinterpret_cast<float*>(a.ws) + at * a.D;
        float* ml = reinterpret_cast<float*>(a.ws) + splits * rows * a.D + at;
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int dd = 32 * d + 8 * i + 4 * h;
                if (dd < a.D) *reinterpret_cast<f32x4*>(op + dd) = f32x4{o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]};
            }
        if (h == 0) { ml[0] = m; ml[splits * rows] = l; }
    }
}

// delta_i = do_i . o_i, one wave per row
template <typename T> __global__ __launch_bounds__(256) void xattn_delta_kernel(sarXattn a, float* delta) {
    const long i = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (i >= (long)a.B * a.Hq * a.Tq) return;
    const int t = (int)(i % a.Tq), hq = (int)(i / a.Tq % a.Hq), b = (int)(i / a.Tq / a.Hq);
    const T* o = reinterpret_cast<const T*>(a.out) + b * a.o_sb + t * a.o_st + hq * a.o_sh;
    const T* g = reinterpret_cast<const T*>(a.dout) + b * a.g_sb + t * a.g_st + hq * a.g_sh;
    float s = 0.f;
    for (int d = threadIdx.x & 63; d < a.D; d += 64) s = fmaf((float)o[d], (float)g[d], s);
    s = wave_sum(s);
    if ((threadIdx.x & 63) == 0) delta[i] = s;
}

// ---- dK, dV: a wave holds 32 keys as columns n (their K and V fragments in registers), the rows stream through LDS
template <typename T, int DP> __global__ __launch_bounds__(256) void xattn_dkv_kernel(sarXattn a, const float* __restrict__ delta, int key_tiles) {
    constexpr int RT = 32, P = pitch<T, DP>(), NC = DP * (int)sizeof(T) / 32, ND = DP / 32;
    __shared__ __attribute__((aligned(16))) char lq[RT * P];
    __shared__ __attribute__((aligned(16))) char lg[RT * P];
    __shared__ __attribute__((aligned(16))) float ls[2][RT];      // lse (in powers of two) and delta of the tile's rows
    const long item = xcd_item((long)a.B * a.Hkv * key_tiles);
    if (item < 0) return;
    const int kt = (int)(item % key_tiles), bh = (int)(item / key_tiles), b = bh / a.Hkv, hk = bh % a.Hkv;
    const int lane = threadIdx.x & 63, h = lane >> 5, n = lane & 31;
    const int len = live_keys(a, b), key0 = kt * 128 + (threadIdx.x >> 6) * 32, key = key0 + n;
    const int rl = kt * 128 < len ? live_rows(a, b) : 0;
    const float sl = a.scale * LOG2E;
    u32x4 kf[NC], vf[NC];
    load_row<T, DP>(reinterpret_cast<const T*>(a.k) + b * a.k_sb + min(key, a.Tk - 1) * a.k_st + hk * a.k_sh, key < len, a.D, h, kf);
    load_row<T, DP>(reinterpret_cast<const T*>(a.v) + b * a.v_sb + min(key, a.Tk - 1) * a.v_st + hk * a.v_sh, key < len, a.D, h, vf);
    const T* qb = reinterpret_cast<const T*>(a.q) + b * a.q_sb;
    const T* gb = reinterpret_cast<const T*>(a.dout) + b * a.g_sb;
    const auto qrow = [&](int r) { const Row w = row_of(a, hk, r); return w.t * a.q_st + w.h * a.q_sh; };
    const auto grow = [&](int r) { const Row w = row_of(a, hk, r); return w.t * a.g_st + w.h * a.g_sh; };
    f32x16 dk[ND], dv[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) { dk[d][i] = 0.f; dv[d][i] = 0.f; }
    Stage<T, DP, RT> sq, sg;
    float st = 0.f;
    const auto load_stats = [&](int r0) {
        if (threadIdx.x < 2 * RT) {
            const int r = r0 + (threadIdx.x & (RT - 1));
            st = threadIdx.x < RT ? INFINITY : 0.f;               // a row that does not exist: p = exp2(s - inf) = 0
            if (r < rl) {
                const long at = stat_at(a, b, row_of(a, hk, r));
                const float v = threadIdx.x < RT ? a.lse[at] * LOG2E : delta[at];
                st = threadIdx.x < RT && v == -INFINITY ? INFINITY : v;
            }
        }
    };
    sq.load(qb, qrow, 0, rl, a.D); sg.load(gb, grow, 0, rl, a.D); load_stats(0);
    for (int r0 = 0; r0 < rl; r0 += RT) {
        __syncthreads();
        sq.store(lq); sg.store(lg);
        if (threadIdx.x < 2 * RT) ls[threadIdx.x / RT][threadIdx.x & (RT - 1)] = st;
        __syncthreads();
        if (r0 + RT < rl) { sq.load(qb, qrow, r0 + RT, rl, a.D); sg.load(gb, grow, r0 + RT, rl, a.D); load_stats(r0 + RT); }
        if (key0 >= len) continue;
        f32x16 s, dp;
#pragma unroll
        for (int i = 0; i < 16; ++i) { s[i] = 0.f; dp[i] = 0.f; }
#pragma unroll
        for (int c = 0; c < NC; ++c) s = mma<T>(frag<P>(lq, n, c, h), kf[c], s);
#pragma unroll
        for (int c = 0; c < NC; ++c) dp = mma<T>(frag<P>(lg, n, c, h), vf[c], dp);
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            const f32x4 e = *reinterpret_cast<const f32x4*>(&ls[0][8 * x + 4 * h]), dl = *reinterpret_cast<const f32x4*>(&ls[1][8 * x + 4 * h]);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const float p = __builtin_amdgcn_exp2f(fmaf(s[4 * x + c], sl, -e[c]));
                s[4 * x + c] = p;
                dp[4 * x + c] = p * (dp[4 * x + c] - dl[c]);
            }
        }
        u32x4 pf[4], df[4];
        pack<T>(s, pf); pack<T>(dp, df);
#pragma unroll
        for (int d = 0; d < ND; ++d) {
            dv[d] = mma_down<T, P>(lg, 0, d, pf, dv[d], lane);
            dk[d] = mma_down<T, P>(lq, 0, d, df, dk[d], lane);
        }
    }
    if (key >= a.Tk) return;
    const bool in = key < len;                                    // frames behind the length: their gradient is zero
    T* kp = reinterpret_cast<T*>(a.dk) + (((long)b * a.Tk + key) * a.Hkv + hk) * a.D;
    T* vp = reinterpret_cast<T*>(a.dv) + (((long)b * a.Tk + key) * a.Hkv + hk) * a.D;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int dd = 32 * d + 8 * i + 4 * h;
            if (dd >= a.D) continue;
            const float f = a.scale;
            store4<T>(kp + dd, in ? dk[d][4 * i] * f : 0.f, in ? dk[d][4 * i + 1] * f : 0.f, in ? dk[d][4 * i + 2] * f : 0.f, in ? dk[d][4 * i + 3] * f : 0.f);
            store4<T>(vp + dd, in ? dv[d][4 * i] : 0.f, in ? dv[d][4 * i + 1] : 0.f, in ? dv[d][4 * i + 2] : 0.f, in ? dv[d][4 * i + 3] : 0.f);
        }
}

// ---- dQ: as the forward, a wave holds 32 rows as columns n, the keys and values stream through LDS
template <typename T, int DP> __global__ __launch_bounds__(256) void xattn_dq_kernel(sarXattn a, const float* __restrict__ delta, int row_tiles) {
    constexpr int KT = 32, P = pitch<T, DP>(), NC = DP * (int)sizeof(T) / 32, ND = DP / 32;
    __shared__ __attribute__((aligned(16))) char lk[KT * P];
    __shared__ __attribute__((aligned(16))) char lv[KT * P];
    const long item = xcd_item((long)a.B * a.Hkv * row_tiles);
    if (item < 0) return;
    const int rt = (int)(item % row_tiles), bh = (int)(item / row_tiles), b = bh / a.Hkv, hk = bh % a.Hkv;
    const int lane = threadIdx.x & 63, h = lane >> 5, n = lane & 31;
    const int R = a.Tq * (a.Hq / a.Hkv), row0 = rt * 128 + (threadIdx.x >> 6) * 32, r = row0 + n;
    const int rl = live_rows(a, b), len = rt * 128 < rl ? live_keys(a, b) : 0;
    const Row me = row_of(a, hk, min(r, R - 1));
    const float sl = a.scale * LOG2E;
    u32x4 qf[NC], gf[NC];
    load_row<T, DP>(reinterpret_cast<const T*>(a.q) + b * a.q_sb + me.t * a.q_st + me.h * a.q_sh, r < rl, a.D, h, qf);
    load_row<T, DP>(reinterpret_cast<const T*>(a.dout) + b * a.g_sb + me.t * a.g_st + me.h * a.g_sh, r < rl, a.D, h, gf);
    float e = r < rl ? a.lse[stat_at(a, b, me)] * LOG2E : INFINITY;
    if (e == -INFINITY) e = INFINITY;
    const float dl = r < rl ? delta[stat_at(a, b, me)] : 0.f;
    const T* kb = reinterpret_cast<const T*>(a.k) + b * a.k_sb + hk * a.k_sh;
    const T* vb = reinterpret_cast<const T*>(a.v) + b * a.v_sb + hk * a.v_sh;
    const auto krow = [&](int j) { return j * a.k_st; };
    const auto vrow = [&](int j) { return j * a.v_st; };
    f32x16 dq[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) dq[d][i] = 0.f;
    Stage<T, DP, KT> sk, sv;
    sk.load(kb, krow, 0, len, a.D); sv.load(vb, vrow, 0, len, a.D);
    for (int j = 0; j < len; j += KT) {
        __syncthreads();
        sk.store(lk); sv.store(lv);
        __syncthreads();
        if (j + KT < len) { sk.load(kb, krow, j + KT, len, a.D); sv.load(vb, vrow, j + KT, len, a.D); }
        if (row0 >= rl) continue;
        f32x16 s, dp;
#pragma unroll
        for (int i = 0; i < 16; ++i) { s[i] = 0.f; dp[i] = 0.f; }
#pragma unroll
        for (int c = 0; c < NC; ++c) s = mma<T>(frag<P>(lk, n, c, h), qf[c], s);
#pragma unroll
        for (int c = 0; c < NC; ++c) dp = mma<T>(frag<P>(lv, n, c, h), gf[c], dp);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const bool in = j + 8 * (i >> 2) + 4 * h + (i & 3) < len;
            const float p = __builtin_amdgcn_exp2f(fmaf(s[i], sl, -e));
            dp[i] = in ? p * (dp[i] - dl) : 0.f;
        }
        u32x4 df[4];
        pack<T>(dp, df);
#pragma unroll
        for (int d = 0; d < ND; ++d) dq[d] = mma_down<T, P>(lk, 0, d, df, dq[d], lane);
    }
    if (r >= R) return;
    T* op = reinterpret_cast<T*>(a.dq) + (((long)b * a.Tq + me.t) * a.Hq + me.h) * a.D;
    const bool in = r < rl;
    const float f = a.scale;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int dd = 32 * d + 8 * i + 4 * h;
            if (dd < a.D)
                store4<T>(op + dd, in ? dq[d][4 * i] * f : 0.f, in ? dq[d][4 * i + 1] * f : 0.f, in ? dq[d][4 * i + 2] * f : 0.f, in ? dq[d][4 * i + 3] * f : 0.f);
        }
}

}  // namespace attn
using namespace attn;

static bool bad(const sarXattn* a) {
    if (bad_shape(a) || bad_strides(sizeof(elt), &a->q_sb, 12)) return true;
    for (const void* p : {a->q, a->k, a->v, (const void*)a->out})
        if (!p || (uintptr_t)p % 16) return true;
    return false;
}

template <int DP> static void launch_fwd(const sarXattn& a, int splits, hipStream_t st) {
    const int rt = cdiv((long)a.Tq * (a.Hq / a.Hkv), 128);
    hipLaunchKernelGGL((xattn_fwd_kernel<elt, DP>), dim3((unsigned)xcd_grid((long)rt * splits * a.B * a.Hkv)), dim3(256), 0, st, a, rt, splits);
}
template <int DP> static void launch_bwd(const sarXattn& a, float* delta, hipStream_t st) {
    const int kt = cdiv(a.Tk, 128), rt = cdiv((long)a.Tq * (a.Hq / a.Hkv), 128);
    hipLaunchKernelGGL((xattn_delta_kernel<elt>), dim3((unsigned)cdiv((long)a.B * a.Hq * a.Tq, 4)), dim3(256), 0, st, a, delta);
    if (kt) hipLaunchKernelGGL((xattn_dkv_kernel<elt, DP>), dim3((unsigned)xcd_grid((long)kt * a.B * a.Hkv)), dim3(256), 0, st, a, delta, kt);
    hipLaunchKernelGGL((xattn_dq_kernel<elt, DP>), dim3((unsigned)xcd_grid((long)rt * a.B * a.Hkv)), dim3(256), 0, st, a, delta, rt);
}

#if SAR_ELT == 0      // the same for every type
extern "C" size_t sar_xattn_fwd_workspace_bytes(const sarXattn* a) { return bad_shape(a) ? 0 : part_bytes(a, few_rows(a) ? step_splits(a) : fwd_splits(a)); }
extern "C" size_t sar_xattn_bwd_workspace_bytes(const sarXattn* a) { return bad_shape(a) ? 0 : 4 * (size_t)a->B * a->Hq * a->Tq; }
#endif

extern "C" int SAR_FN(sar_xattn_fwd)(const sarXattn* a, hipStream_t stream) {
    if (bad(a)) return SAR_EINVAL;
    if (bad_workspace(a, part_bytes(a, few_rows(a) ? step_splits(a) : fwd_splits(a)))) return SAR_EINVAL;
    if (few_rows(a)) return SAR_FN(xattn_step)(a, step_splits(a), stream);
    const int splits = fwd_splits(a);
    if (a->D <= 32) launch_fwd<32>(*a, splits, stream);
    else if (a->D <= 64) launch_fwd<64>(*a, splits, stream);
    else if (a->D <= 96) launch_fwd<96>(*a, splits, stream);
    else launch_fwd<128>(*a, splits, stream);
    SAR_CHECK_LAUNCH();
    return splits > 1 ? SAR_FN(xattn_combine)(a, splits, stream) : SAR_OK;
}

extern "C" int SAR_FN(sar_xattn_bwd)(const sarXattn* a, hipStream_t stream) {
    if (bad(a) || !a->lse || !a->dout || !a->dq || !a->dk || !a->dv || !a->ws) return SAR_EINVAL;
    for (const void* p : {a->dout, (const void*)a->dq, (const void*)a->dk, (const void*)a->dv})
        if ((uintptr_t)p % 16) return SAR_EINVAL;
    if (bad_strides(sizeof(elt), &a->g_sb, 3) || bad_workspace(a, 4 * (size_t)a->B * a->Hq * a->Tq)) return SAR_EINVAL;
    float* delta = reinterpret_cast<float*>(a->ws);
    if (a->D <= 32) launch_bwd<32>(*a, delta, stream);
    else if (a->D <= 64) launch_bwd<64>(*a, delta, stream);
    else if (a->D <= 96) launch_bwd<96>(*a, delta, stream);
    else launch_bwd<128>(*a, delta, stream);
    SAR_CHECK_LAUNCH();
    return SAR_OK;
}
