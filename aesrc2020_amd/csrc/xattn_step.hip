// Attention of a FEW rows (one token, a beam's tokens) to many keys: up to 32 folded rows (tokens x query heads of a key head) are the
// columns n of one MFMA tile, every wave of a block walks its own 32-key tiles without a barrier, waves and key slices are joined at the end.
// Reading the keys and values once is the whole cost, so what counts is bytes in flight: a wave has two buffers for a K and a V tile in LDS and
// loads the next tile straight into one (whole rows, coalesced) while it computes from the other.
//
// The same kernel reads the 8-bit cache (include/sarnet.h: sarKv8): e4m3 values are converted exactly into the 16-bit operand type (bf16 for
// bf16 and fp32 queries, fp16 for fp16 ones); the scale of a 64-key block multiplies the fp32 scores (K); V's goes into the bf16 values (a bf16 has
// an fp32's range), and beside fp16 ones into the fp32 sums as a ratio of powers of two.  fp32 queries and probabilities enter as three bf16
// planes (8 + 8 + 8 bits hold an fp32 mantissa): products are exact, sums fp32, at a third of the bf16 rate instead of the fp32 MFMA's sixteenth.
// Compiled once per element type: SAR_ELT 0 = fp32, 1 = bf16, 2 = fp16.
#include "xattn.h"

#if SAR_ELT == 0
typedef float elt;
typedef __bf16 wide8;
#define SAR_FN(n) n##_f32
#elif SAR_ELT == 1
typedef __bf16 elt;
typedef __bf16 wide8;
#define SAR_FN(n) n##_bf16
#else
typedef _Float16 elt;
typedef _Float16 wide8;
#define SAR_FN(n) n##_f16
#endif

namespace attn {

constexpr int KV_BLOCK = 64;            // frames that share a scale

struct Kv8 { const unsigned char *k8, *v8; const float *ks, *vs; long frames; };   // (B, Hkv, frames, D), (B, Hkv, frames / 64)

// eight e4m3 values times a power of two -> eight 16-bit ones, exactly
template <typename C> __device__ __forceinline__ u32x4 widen8(u32x2 w, float scale) {
    u32x4 o;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int src = (int)w[i >> 1];
        if constexpr (__is_same(C, __bf16)) {
            const auto v = (i & 1) ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(src, scale, true) : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(src, scale, false);
            o[i] = __builtin_bit_cast(unsigned, v);
        } else {
            const auto v = (i & 1) ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(src, scale, true) : __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(src, scale, false);
            o[i] = __builtin_bit_cast(unsigned, v);
        }
    }
    return o;
}
// mma_down (attn_tiles.h) over a tile of e4m3 rows: the transposing read hands a lane eight rows of one column as bytes
template <typename C, int PITCH> __device__ __forceinline__ u32x4 down8(const char* tile, int dt, int s, int lane, float scale) {
    const int i = lane & 15, slot = i >> 1, r = 16 * s + 4 * (lane >> 5) + (slot & 3) + 8 * (slot >> 2);
    typedef __attribute__((ext_vector_type(2))) int i32x2;
    const i32x2 v = __builtin_amdgcn_ds_read_tr8_b64_v2i32((__attribute__((address_space(3))) i32x2*)(tile + chunk_at<PITCH>(r, 2 * dt + ((lane >> 4) & 1)) + (i & 1) * 8));
    return widen8<C>(__builtin_bit_cast(u32x2, v), scale);
}

// a 32 x 32 fp32 result as operand planes of the 16-bit type: one (rounded), or three whose sum is the value
template <typename C, int NPL> __device__ __forceinline__ void pack_planes(f32x16 s, u32x4 (*p)[4]) {
#pragma unroll
    for (int k = 0; k < NPL; ++k) {
        pack<C>(s, p[k]);
        if (k + 1 < NPL)
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] -= (float)(C)s[i];
    }
}

template <typename T, bool S8, int DP> constexpr int step_pitch() { return S8 ? (DP <= 64 ? 64 : 128) : pitch<T, DP>(); }
// waves of a block: each has two buffers of a K and a V tile (128 KB of LDS at most); narrow rows leave room for eight
template <typename T, bool S8, int DP> constexpr int step_waves() { return step_pitch<T, S8, DP>() <= 256 ? 4 : 2; }
template <typename T, bool S8, int DP> constexpr int most_waves() { return step_pitch<T, S8, DP>() <= 128 ? 8 : step_waves<T, S8, DP>(); }

template <typename T, typename C, bool S8, int DP, int NW> __global__ __launch_bounds__(64 * NW, 2) void xattn_step_kernel(sarXattn a, Kv8 kv, int row_tiles, int splits) {
    constexpr int P = step_pitch<T, S8, DP>(), ND = DP / 32, NPL = S8 && sizeof(T) == 4 ? 3 : 1, TILE = 32 * P;
    constexpr int NC = DP * (int)sizeof(C) / 32;                  // operand chunks of a row
    typedef WaveLoader<P> Loader;
    extern __shared__ __attribute__((aligned(1024))) char lds[];  // K and V tiles of the waves; afterwards their partial sums
    __shared__ float lm[NW][32], ll[NW][32];
    const int item = xcd_item(a.B * a.Hkv * row_tiles * splits);
    if (item < 0) return;
    const int sp = item % splits, rt = item / splits % row_tiles, bh = item / splits / row_tiles;
    const int b = bh / a.Hkv, hk = bh % a.Hkv;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, h = lane >> 5, n = lane & 31;
    const int R = a.Tq * (a.Hq / a.Hkv), r = rt * 32 + n, rl = live_rows(a, b), len = live_keys(a, b);
    const int tiles = (len + 31) / 32, per = (tiles + splits - 1) / splits;
    const int t0 = min(sp * per, tiles), t1 = rt * 32 < rl ? min(t0 + per, tiles) : t0;
    const Row me = row_of(a, hk, min(r, R - 1));
    const float sl = score_factor(a);                             // (the scale's sign is in the queries: xattn.hip)
    const bool negate = a.scale < 0.f;

    const unsigned bytes = (unsigned)(a.D * (S8 ? 1 : (int)sizeof(T)));
    const long k_st = S8 ? a.D : a.k_st * (long)sizeof(T), v_st = S8 ? a.D : a.v_st * (long)sizeof(T);
    const char* kb = S8 ? reinterpret_cast<const char*>(kv.k8) + (long)bh * kv.frames * a.D : reinterpret_cast<const char*>(a.k) + (b * a.k_sb + hk * a.k_sh) * (long)sizeof(T);
    const char* vb = S8 ? reinterpret_cast<const char*>(kv.v8) + (long)bh * kv.frames * a.D : reinterpret_cast<const char*>(a.v) + (b * a.v_sb + hk * a.v_sh) * (long)sizeof(T);
    // (scalar loads: a vector load among the tile loads would be waited for with them)
    typedef const __attribute__((address_space(4))) float* scales;
    const scales ks = S8 ? (scales)(uintptr_t)(kv.ks + (long)bh * (kv.frames / KV_BLOCK)) : nullptr, vs = S8 ? (scales)(uintptr_t)(kv.vs + (long)bh * (kv.frames / KV_BLOCK)) : nullptr;
    const Loader lk((unsigned)k_st), lv((unsigned)v_st);
    char* mine = lds + w * 4 * TILE;
    const unsigned to = lds_addr(mine);
    const auto load = [&](int t, int buf) {
        lk.load(kb + t * 32 * k_st, len - t * 32, (unsigned)k_st, bytes, to + buf);
        lv.load(vb + t * 32 * v_st, len - t * 32, (unsigned)v_st, bytes, to + buf + TILE);
    };
    if (t0 + w < t1) load(t0 + w, 0);

    u32x4 qf[NPL][NC];
    {
        const T* qp = reinterpret_cast<const T*>(a.q) + b * a.q_sb + me.t * a.q_st + me.h * a.q_sh;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            // the order of the dims among the contraction's slots follows the stored keys: 16 bytes a lane and half
            const int d = S8 ? 32 * (c >> 1) + 16 * h + 8 * (c & 1) : (2 * c + h) * Num<T>::PER;
            const bool ok = r < rl && d < a.D;
            if constexpr (S8 && sizeof(T) == 4) {
                f32x4 x0 = {0, 0, 0, 0}, x1 = {0, 0, 0, 0};
                if (ok) { x0 = *reinterpret_cast<const f32x4*>(qp + d); x1 = *reinterpret_cast<const f32x4*>(qp + d + 4); }
                if (negate) { x0 = -x0; x1 = -x1; }
#pragma unroll
                for (int k = 0; k < NPL; ++k) {
                    typename Num<C>::x16 v;
#pragma unroll
                    for (int j = 0; j < 4; ++j) { v[j] = (C)x0[j]; v[4 + j] = (C)x1[j]; x0[j] -= (float)v[j]; x1[j] -= (float)v[4 + j]; }
                    qf[k][c] = __builtin_bit_cast(u32x4, v);
                }
            } else {
                qf[0][c] = u32x4{0, 0, 0, 0};
                if (ok) qf[0][c] = *reinterpret_cast<const u32x4*>(qp + d);
                if (negate) qf[0][c] = qf[0][c] ^ (sizeof(T) == 4 ? 0x80000000u : 0x80008000u);
            }
        }
    }
    f32x16 o[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[d][i] = 0.f;
    // fp16 values of a cache: o holds sums in units of V's scale, `unit`, else 1.  (A block whose values end below 2^-31 counts as one of that size:
    // no fp16 result shows it.)
    constexpr bool UNITS = S8 && __is_same(C, _Float16);
    constexpr float MOST = 3.4028235e38f;
    const auto unit_of = [&](int t) { return fmaxf(vs[t * 32 / KV_BLOCK], 9.094947017729282e-13f); };
    float m = NO_MAX, l = 0.f, unit = 1.f;
    if (UNITS && t0 + w < t1) unit = unit_of(t0 + w);
    bool large = false;
    int cur = 0;
    for (int t = t0 + w; t < t1; t += NW, cur ^= 2 * TILE) {
        if (t + NW < t1) {
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");    // the reads of the buffer that is loaded next are done
            load(t + NW, cur ^ (2 * TILE));
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * Loader::N) : "memory");
        } else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        const char *tk = mine + cur, *tv = tk + TILE;
        f32x16 tile_s[1], &s = tile_s[0];
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = 0.f;
        if constexpr (S8) {
#pragma unroll
            for (int c = 0; c < DP / 32; ++c) {
                u32x4 x = frag<P>(tk, n, c, h);
                if (a.D & 8) {                                    // a row ends inside a piece: what follows is the next row
                    const bool half = 32 * c + 16 * h + 8 >= a.D;
                    x[2] = half ? 0 : x[2]; x[3] = half ? 0 : x[3];
                }
                const u32x4 lo = widen8<C>(u32x2{x[0], x[1]}, 1.f), hi = widen8<C>(u32x2{x[2], x[3]}, 1.f);
#pragma unroll
                for (int k = NPL - 1; k >= 0; --k) { s = mma<C>(lo, qf[k][2 * c], s); s = mma<C>(hi, qf[k][2 * c + 1], s); }
            }
        } else {
#pragma unroll
            for (int c = 0; c < NC; ++c) s = mma<T>(frag<P>(tk, n, c, h), qf[0][c], s);
        }
        const float f = S8 ? fmaxf(fabsf(a.scale) * LOG2E * ks[t * 32 / KV_BLOCK], LEAST) : sl, nu = UNITS ? unit_of(t) : 1.f, v_scale = S8 && !UNITS ? vs[t * 32 / KV_BLOCK] : 1.f;
        float top = NO_MAX;
        if (t * 32 + 32 > len) {
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = t * 32 + 8 * (i >> 2) + 4 * h + (i & 3) < len ? s[i] : -INFINITY;
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) top = fmaxf(top, s[i]);
        top = half_max(top) * f;
        if (__any(top - m > lag<C>()) || (UNITS && nu != unit)) {
            const float mn = fmaxf(m, reference<C>(top)), e = __builtin_amdgcn_exp2f(m - mn);
            const float eo = UNITS ? fminf(e * unit / nu, MOST) : e;             // (in this order: no power of two passes the range before e has taken it back)
            const bool beyond = UNITS && unit > nu * 1.2089258196146292e24f;     // by 2^80: sums other than 0 are past fp16's range, and stay finite here
            m = mn; l *= e;
            large = __any(fabsf(m) > LARGE && m != NO_MAX);
            if (UNITS) unit = nu;
#pragma unroll
            for (int d = 0; d < ND; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[d][i] *= eo;
            if (UNITS && __builtin_expect(beyond, 0)) {
#pragma unroll
                for (int d = 0; d < ND; ++d)
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[d][i] = fabsf(o[d][i]) == INFINITY ? copysignf(MOST, o[d][i]) : o[d][i];
            }
        }
        exponents(tile_s, f, m, large);
#pragma unroll
        for (int i = 0; i < 16; ++i) { s[i] = __builtin_amdgcn_exp2f(s[i]); l += s[i]; }
        u32x4 p[NPL][4];
        pack_planes<C, NPL>(s, p);
#pragma unroll
        for (int d = 0; d < ND; ++d) {
            if constexpr (S8) {
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const u32x4 v = down8<C, P>(tv, d, x, lane, v_scale);
#pragma unroll
                    for (int k = NPL - 1; k >= 0; --k) o[d] = mma<C>(v, p[k][x], o[d]);
                }
            } else o[d] = mma_down<C, P>(tv, 0, d, p[0], o[d], lane);
        }
    }
    l = half_sum(l);

    // ---- join the waves: o, m, l of the live rows through LDS
    const int nr = min(R - rt * 32, 32);
    float* lo = reinterpret_cast<float*>(lds);
    __syncthreads();                                              // every wave is done with its V tile
    if (n < nr) {
        float* op = lo + ((long)w * nr + n) * DP;
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                *reinterpret_cast<f32x4*>(op + 32 * d + 8 * i + 4 * h) = f32x4{o[d][4 * i] * unit, o[d][4 * i + 1] * unit, o[d][4 * i + 2] * unit, o[d][4 * i + 3] * unit};
        if (h == 0) { lm[w][n] = m; ll[w][n] = l; }
    }
    __syncthreads();
    const int D4 = a.D / 4;
    for (int e = threadIdx.x; e < nr * D4; e += 64 * NW) {
        const int row = e / D4, d = (e - row * D4) * 4;
        float M = lm[0][row];
#pragma unroll
        for (int x = 1; x < NW; ++x) M = fmaxf(M, lm[x][row]);
        float L = 0.f;
        f32x4 v = {0, 0, 0, 0};
#pragma unroll
        for (int x = 0; x < NW; ++x) {
            const float g = __builtin_amdgcn_exp2f(lm[x][row] - M);
            L = fmaf(ll[x][row], g, L);
            v += *reinterpret_cast<const f32x4*>(lo + ((long)x * nr + row) * DP + d) * g;
        }
        const Row at = row_of(a, hk, rt * 32 + row);
        if (splits == 1) {
            const bool in = rt * 32 + row < rl && L != 0.f;
            const float inv = 1.f / L;
            store4<T>(reinterpret_cast<T*>(a.out) + b * a.o_sb + at.t * a.o_st + at.h * a.o_sh + d, in ? v[0] * inv : 0.f, in ? v[1] * inv : 0.f, in ? v[2] * inv : 0.f, in ? v[3] * inv : 0.f);
            if (a.lse && d == 0) a.lse[stat_at(a, b, at)] = in ? M * LN2 + logf(L) : -INFINITY;
        } else {
            const long rows = (long)a.B * a.Hq * a.Tq, i = sp * rows + stat_at(a, b, at);
            *reinterpret_cast<f32x4*>(reinterpret_cast<float*>(a.ws) + i * a.D + d) = v;
            if (d == 0) {
                float* ml = reinterpret_cast<float*>(a.ws) + splits * rows * a.D + i;
                ml[0] = M; ml[splits * rows] = L;
            }
        }
    }
}

// joins the key slices: one wave per row
template <typename T> __global__ __launch_bounds__(256) void xattn_combine_kernel(sarXattn a, int splits) {
    const long rows = (long)a.B * a.Hq * a.Tq, i = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (i >= rows) return;
    const int t = (int)(i % a.Tq), hq = (int)(i / a.Tq % a.Hq), b = (int)(i / a.Tq / a.Hq), lane = threadIdx.x & 63;
    const float* po = reinterpret_cast<const float*>(a.ws);
    const float* pm = po + splits * rows * a.D;
    const float m = lane < splits ? pm[lane * rows + i] : NO_MAX, l = lane < splits ? pm[(splits + lane) * rows + i] : 0.f;
    const float M = wave_max(m), f = __builtin_amdgcn_exp2f(m - M), L = wave_sum(l * f);
    const bool in = t < (a.q_lens ? min(max(a.q_lens[b], 0), a.Tq) : a.Tq) && L != 0.f;
    const int d = 2 * lane;
    float x = 0.f, y = 0.f;
    for (int s = 0; s < splits; ++s) {
        const float g = __shfl(f, s, 64);
        if (d < a.D) {
            const float2 v = *reinterpret_cast<const float2*>(po + (s * rows + i) * a.D + d);
            x = fmaf(v.x, g, x); y = fmaf(v.y, g, y);
        }
    }
    const float inv = 1.f / L;
    if (d < a.D) {
        T* op = reinterpret_cast<T*>(a.out) + b * a.o_sb + t * a.o_st + hq * a.o_sh + d;
        op[0] = (T)(in ? x * inv : 0.f); op[1] = (T)(in ? y * inv : 0.f);
    }
    if (a.lse && lane == 0) a.lse[i] = in ? M * LN2 + logf(L) : -INFINITY;
}

// a launch has fewer than 2^32 threads along an axis: blocks in rows of so many
constexpr int LAUNCH_ROW = 1 << 22;
// ---- writing the cache: one block per (K or V, utterance, head, 64 frames): maximum, scale, conversion in one pass over its 64 D values
struct Kv8Side { const void* x; long sb, st, sh; unsigned char* y; float* scale; };
template <typename T> __global__ __launch_bounds__(256) void kv8_store_kernel(Kv8Side sk, Kv8Side sv, const int* __restrict__ lens, int* __restrict__ lens_out, int T_in, int H, int D,
                                                                              long frames, int first, unsigned blocks, unsigned total) {
    __shared__ float red[4];
    constexpr int V = 8;                                          // values a thread and step; D is a multiple of 8
    const Kv8Side& sd = blockIdx.y ? sv : sk;
    const T* x = reinterpret_cast<const T*>(sd.x);
    const long sb = sd.sb, st = sd.st, sh = sd.sh;
    const unsigned item = min(blockIdx.x + LAUNCH_ROW * blockIdx.z, total - 1);    // (the last row's surplus blocks write the last item's values again)
    const int j = item % blocks, bh = item / blocks, b = bh / H, hh = bh % H;
    const int per = D / V, n = KV_BLOCK * per;                    // <= 1024: four steps
    const int live = lens ? min(max(lens[b], 0), T_in) : T_in;
    // the cache's length: an utterance without new frames keeps the one it has
    if (j == 0 && hh == 0 && blockIdx.y == 0 && threadIdx.x == 0 && (live > 0 || first == 0)) lens_out[b] = first + live;
    float v[4][V];
    float top = 0.f;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
        const int e = threadIdx.x + 256 * s, row = e / per, d = (e - row * per) * V, t = j * KV_BLOCK + row;
#pragma unroll
        for (int k = 0; k < V; ++k) v[s][k] = 0.f;
        if (e < n && t < live) {
            const T* p = x + b * sb + (long)t * st + hh * sh + d;
#pragma unroll
            for (int q = 0; q < V; q += Num<T>::PER) {
                const auto u = *reinterpret_cast<const typename Num<T>::x16*>(p + q);
#pragma unroll
                for (int k = 0; k < Num<T>::PER; ++k) v[s][q + k] = (float)u[k];
            }
#pragma unroll
            for (int k = 0; k < V; ++k) { const float m = fabsf(v[s][k]); if (m < INFINITY) top = fmaxf(top, m); }
        }
    }
    top = wave_max(top);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = top;
    __syncthreads();
    top = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    // top = f 2^e, f in [1/2, 1): the smallest power of two with top / scale <= 448 = 7/8 2^9.  (Held at 2^-118 and above: its inverse stays finite.)
    int e = 0;
    const float f = frexpf(top, &e);
    e = top == 0.f ? 0 : max(f <= 0.875f ? e - 9 : e - 8, -118);
    const float inv = ldexpf(1.f, -e);
    const long blk = (long)bh * (frames / KV_BLOCK) + first / KV_BLOCK + j;
    if (threadIdx.x == 0) sd.scale[blk] = ldexpf(1.f, e);
    unsigned char* o = sd.y + blk * KV_BLOCK * D;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
        const int q = threadIdx.x + 256 * s;
        if (q >= n) continue;
        u32x2 w;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            int p = 0;
            p = __builtin_amdgcn_cvt_pk_fp8_f32(v[s][4 * k] * inv, v[s][4 * k + 1] * inv, p, false);
            p = __builtin_amdgcn_cvt_pk_fp8_f32(v[s][4 * k + 2] * inv, v[s][4 * k + 3] * inv, p, true);
            w[k] = (unsigned)p;
        }
        *reinterpret_cast<u32x2*>(o + (long)q * V) = w;
    }
}

}  // namespace attn
using namespace attn;

int SAR_FN(xattn_combine)(const sarXattn* a, int splits, hipStream_t stream);

template <typename C, bool S8, int DP, int NW> static int launch_waves(const sarXattn& a, const Kv8& kv, int splits, hipStream_t st) {
    const long R = (long)a.Tq * (a.Hq / a.Hkv);
    const int rt = cdiv(R, 32);
    const size_t tiles = (size_t)NW * 4 * 32 * step_pitch<elt, S8, DP>(), join = (size_t)NW * (R < 32 ? R : 32) * DP * 4, lds = tiles > join ? tiles : join;
    auto* k = &xattn_step_kernel<elt, C, S8, DP, NW>;
    static PerDeviceFlag raised;
    if (lds > 64 * 1024 && !raised) {
        if (hipFuncSetAttribute(reinterpret_cast<const void*>(k), hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024 - 4096) != hipSuccess) return SAR_ELAUNCH;
        raised = true;
    }
    hipLaunchKernelGGL(k, dim3((unsigned)xcd_grid((long)rt * splits * a.B * a.Hkv)), dim3(64 * NW), lds, st, a, kv, rt, splits);
    SAR_CHECK_LAUNCH();
    return SAR_OK;
}
// without key slices, the wider block where the keys are many for four waves
template <typename C, bool S8, int DP> static int launch_step(const sarXattn& a, const Kv8& kv, hipStream_t st) {
    constexpr int NW = step_waves<elt, S8, DP>(), MW = most_waves<elt, S8, DP>();
    const int splits = step_splits(&a, MW, SAR_ELT == 0);
    if (bad_workspace(&a, part_bytes(&a, splits))) return SAR_EINVAL;
    if constexpr (MW > NW) {
        if (splits == 1 && a.Tk > 256) return launch_waves<C, S8, DP, MW>(a, kv, 1, st);
    }
    const int rc = launch_waves<C, S8, DP, NW>(a, kv, splits, st);
    return rc == SAR_OK && splits > 1 ? SAR_FN(xattn_combine)(&a, splits, st) : rc;
}

int SAR_FN(xattn_combine)(const sarXattn* a, int splits, hipStream_t stream) {
    hipLaunchKernelGGL((xattn_combine_kernel<elt>), dim3((unsigned)cdiv((long)a->B * a->Hq * a->Tq, 4)), dim3(256), 0, stream, *a, splits);
    SAR_CHECK_LAUNCH();
    return SAR_OK;
}

template <typename C, bool S8> static int step(const sarXattn* a, const Kv8& kv, hipStream_t stream) {
    return a->D <= 32 ? launch_step<C, S8, 32>(*a, kv, stream) : a->D <= 64 ? launch_step<C, S8, 64>(*a, kv, stream)
         : a->D <= 96 ? launch_step<C, S8, 96>(*a, kv, stream) : launch_step<C, S8, 128>(*a, kv, stream);
}
int SAR_FN(xattn_step)(const sarXattn* a, hipStream_t stream) { return step<elt, false>(a, Kv8{}, stream); }

// ---- the 8-bit cache
static bool bad8(const sarXattn* a, long frames) { return bad_shape(a) || frames < a->Tk || frames % KV_BLOCK || frames > (1L << 30); }
#if SAR_ELT == 0      // the same for every type
extern "C" size_t sar_kv8_attend_workspace_bytes(const sarXattn* a) {            // (its rows are at most 128 bytes: eight waves)
    return bad_shape(a) ? 0 : part_bytes(a, step_splits(a, 8, a->elt_bytes != 2));
}
#endif
extern "C" int SAR_FN(sar_kv8_attend)(const sarXattn* a, const void* k8, const float* k_scale, const void* v8, const float* v_scale, long frames, hipStream_t stream) {
    if (bad8(a, frames) || bad_strides(sizeof(elt), &a->q_sb, 3) || bad_strides(sizeof(elt), &a->o_sb, 3) || !a->q || !a->out || !k8 || !v8 || !k_scale || !v_scale) return SAR_EINVAL;
    for (const void* p : {a->q, (const void*)a->out, k8, v8})
        if ((uintptr_t)p % 16) return SAR_EINVAL;
    return step<wide8, true>(a, Kv8{(const unsigned char*)k8, (const unsigned char*)v8, k_scale, v_scale, frames}, stream);
}
extern "C" int SAR_FN(sar_kv8_store)(const void* k, long k_sb, long k_st, long k_sh, const void* v, long v_sb, long v_st, long v_sh, const int* lens, void* k8, float* k_scale,
                                     void* v8, float* v_scale, int* lens_out, int B, int T, int H, int D, long frames, int first, hipStream_t stream) {
    const long s[6] = {k_sb, k_st, k_sh, v_sb, v_st, v_sh};
    if (bad_strides(sizeof(elt), s, 6) || !k_scale || !v_scale || !lens_out || B < 1 || T < 1 || H < 1 || D < 8 || D > 128 || D % 8 || frames % KV_BLOCK || frames > (1L << 30) ||
        first < 0 || first % KV_BLOCK || first + (long)T > frames)
        return SAR_EINVAL;
    for (const void* p : {k, v, (const void*)k8, (const void*)v8})
        if (!p || (uintptr_t)p % 16) return SAR_EINVAL;
    const int blocks = cdiv(T, KV_BLOCK);
    if ((long)B * H > (1L << 30) / blocks) return SAR_EINVAL;
    const int total = B * H * blocks;
    const Kv8Side ks = {k, k_sb, k_st, k_sh, (unsigned char*)k8, k_scale}, vs = {v, v_sb, v_st, v_sh, (unsigned char*)v8, v_scale};
    const int row = total < LAUNCH_ROW ? total : LAUNCH_ROW;
    hipLaunchKernelGGL((kv8_store_kernel<elt>), dim3((unsigned)row, 2, (unsigned)cdiv(total, row)), dim3(256), 0, stream, ks, vs, lens, lens_out, T, H, D, frames, first, (unsigned)blocks,
                       (unsigned)total);
    SAR_CHECK_LAUNCH();
    return SAR_OK;
}
