// Softmax cross entropy over a vocabulary straight from the hidden rows and the output layer's (D, V) kernel, without a (R, V) array of
// logits or probabilities.
//
//   z = x W + b    lse_r = log sum_v exp z_rv    loss_r = lse_r - z_{r, label}    (0 for a label outside [0, V))
//   dz_rv = g_r (exp(z_rv - lse_r) - [v = label_r])    dx = dz W^T    dW = x^T dz    db = sum_r dz
//
// Forward: one product whose epilogue keeps the maximum and the sum of every 64 vocabulary entries of a row; a small kernel joins them.
// Backward, in pieces of the vocabulary: the piece's logits are computed again, turned into dz in the epilogue and written once in the
// operand type; two more products read that piece (it stays in the last-level cache) for dx and dW.
//
// All products run on the 32x32x16 matrix instructions.  fp32 operands are two fp16 planes under one power-of-two scale per tensor that puts its
// largest element in [2^13, 2^14): hi + lo hold 22 bits, hi hi + hi lo + lo hi is the product to 2^-22 or so of |a| |b|, at a third of the fp16 rate
// (the fp32 matrix instructions run at a sixteenth).  dz is scaled by the power of two that puts the largest |g| in (1/2, 1], times 2^14:
// every probability down to 2^-28 is a normal fp16 number.
// Compiled once per element type: SAR_ELT 0 = fp32, 1 = bf16, 2 = fp16.
#include "attn_tiles.h"

#if SAR_ELT == 0
typedef float elt;
typedef _Float16 op16;
#define SAR_FN(n) n##_f32
#define SAR_WS(n) n##_f32_workspace_bytes
#elif SAR_ELT == 1
typedef __bf16 elt;
typedef __bf16 op16;
#define SAR_FN(n) n##_bf16
#define SAR_WS(n) n##_bf16_workspace_bytes
#else
typedef _Float16 elt;
typedef _Float16 op16;
#define SAR_FN(n) n##_f16
#define SAR_WS(n) n##_f16_workspace_bytes
#endif

// include/sarnet.h: sarVocabCe (kept field for field)
struct sarVocabCe {
    const void *x, *kernel, *bias, *labels;
    const float* dloss;
    float *loss, *lse;
    void *dx, *dkernel, *dbias;
    void* ws;
    long ws_bytes;
    long ldx, ldk;
    int R, D, V, label_bytes, accumulate, pad_;
};

// one namespace per build: the templates below differ from build to build under the same arguments
namespace SAR_FN(vce) {
using attn::Num;
using attn::chunk_at;
using attn::as16;

constexpr float LOG2E = 1.4426950408889634f;
constexpr int BK = 32;                  // contraction elements per LDS stage
constexpr int NPL = SAR_ELT == 0 ? 2 : 1;
constexpr int PAIRS = NPL == 2 ? 3 : 1;
constexpr int DZ_BITS = 14;

// Device scalars of a call: maxima of |x|, |W| (fp32 only) and |dloss|, reduced from 256 partial maxima each by whoever reads them
constexpr int PARTS = 256;
__device__ __forceinline__ float max_of(const float* part) {
    const int l = threadIdx.x & 63;
    return wave_max(fmaxf(fmaxf(part[l], part[l + 64]), fmaxf(part[l + 128], part[l + 192])));
}
// exponent e with v 2^e in [2^13, 2^14) (0 for v = 0), kept where 2^e and 2^-e are ordinary numbers
__device__ __forceinline__ int up_exp(float v) {
    int e = 0;
    (void)frexpf(v, &e);
    return v == 0.f ? 0 : min(max(14 - e, -110), 110);
}
__device__ __forceinline__ int g_exp(float v) {                   // v 2^-e in [1/2, 1)
    int e = 0;
    (void)frexpf(v, &e);
    return v == 0.f ? 0 : min(max(e, -110), 110);
}

template <typename T> __global__ __launch_bounds__(256) void absmax_kernel(const T* __restrict__ x, long rows, int cols, long ld, float* __restrict__ part) {
    __shared__ float red[16];
    float m = 0.f;
    for (long r = blockIdx.x; r < rows; r += gridDim.x)
        for (int c = threadIdx.x; c < cols; c += 256) {
            const float v = fabsf((float)x[r * ld + c]);
            if (v < INFINITY) m = fmaxf(m, v);
        }
    m = block_max(m, red);
    if (threadIdx.x == 0) part[blockIdx.x] = m;
    if (blockIdx.x == 0)                                          // fewer blocks than PARTS: the others' places
        for (int i = gridDim.x + threadIdx.x; i < PARTS; i += 256) part[i] = 0.f;
}

// rows of `cols` elements -> rows of `pitch` operand elements, zeros behind (planes hi, lo for fp32)
template <typename T> __global__ __launch_bounds__(256) void pack_kernel(const T* __restrict__ x, long rows, int cols, long ld, op16* __restrict__ y, long plane, int pitch, const float* __restrict__ part) {
    const float f = NPL == 2 ? ldexpf(1.f, up_exp(max_of(part))) : 1.f;
    const long n = rows * (pitch / 8);
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long)gridDim.x * 256) {
        const long r = i / (pitch / 8);
        const int c = (int)(i - r * (pitch / 8)) * 8;
        typename Num<op16>::x16 hi, lo;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const T v = c + k < cols ? x[r * ld + c + k] : (T)0.f;
            if constexpr (NPL == 2) {
                const float s = (float)v * f;
                hi[k] = (op16)s;
                lo[k] = (op16)(s - (float)hi[k]);
            } else hi[k] = v;
        }
        *reinterpret_cast<typename Num<op16>::x16*>(y + r * pitch + c) = hi;
        if constexpr (NPL == 2) *reinterpret_cast<typename Num<op16>::x16*>(y + plane + r * pitch + c) = lo;
    }
}

// One operand of a product: `len` rows or columns (the output's side), contraction length k.
// DOWN = false: element (i, k) at p[i ld + k] (k contiguous).  DOWN = true: element (i, k) at p[k ld + i] (read down the columns).
struct Side { const op16* p; long plane, ld; int len, k; };

template <int ROWS, bool DOWN> struct Loader {
    static constexpr int N = ROWS * BK * 2 / 16 / 256;            // 16-byte chunks per thread and stage
    u32x4 r[N];
    __device__ __forceinline__ void load(const Side& s, const op16* base, int i0, int k0) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int idx = threadIdx.x + 256 * j;
            if constexpr (DOWN) {
                // rows behind the contraction's end meet zeros of the other operand: any row of the tensor will do; columns behind the output's
                // end are results nobody writes
                const int k = min(k0 + idx / (ROWS / 8), s.k - 1), i = min(i0 + idx % (ROWS / 8) * 8, s.len - 8);
                r[j] = *reinterpret_cast<const u32x4*>(base + k * s.ld + i);
            } else {
                const int i = min(i0 + idx / 4, s.len - 1);
                r[j] = *reinterpret_cast<const u32x4*>(base + i * s.ld + k0 + idx % 4 * 8);
            }
        }
    }
    __device__ __forceinline__ void store(char* tile) const {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int idx = threadIdx.x + 256 * j;
            if constexpr (DOWN) *reinterpret_cast<u32x4*>(tile + chunk_at<ROWS * 2>(idx / (ROWS / 8), idx % (ROWS / 8))) = r[j];
            else *reinterpret_cast<u32x4*>(tile + chunk_at<BK * 2>(idx / 4, idx % 4)) = r[j];
        }
    }
};
// operand fragment: 32 rows at i0, sixteen contraction elements at 16 s
template <int ROWS, bool DOWN> __device__ __forceinline__ u32x4 fragment(const char* tile, int i0, int s, int lane) {
    if constexpr (DOWN) {
        const int i = lane & 15, k = 16 * s + 8 * (lane >> 5) + (i >> 2), ch = (i0 >> 3) + 2 * ((lane >> 4) & 1) + ((i >> 1) & 1), off = (i & 1) * 8;
        const u32x2 a = attn::tr16(tile + chunk_at<ROWS * 2>(k, ch) + off), b = attn::tr16(tile + chunk_at<ROWS * 2>(k + 4, ch) + off);
        return u32x4{a[0], a[1], b[0], b[1]};
    } else return *reinterpret_cast<const u32x4*>(tile + chunk_at<BK * 2>(i0 + (lane & 31), 2 * s + (lane >> 5)));
}

// what happens to a finished tile: C (m, n), column n = lane % 32 of a 32 x 32 tile
enum { E_LSE, E_DZ, E_OUT, E_PART };
struct Epi {
    const float *part_x, *part_w, *part_g;       // exponents (fp32: x, W; gradients: dloss)
    const elt* bias;
    const void* labels;
    const float *dloss, *lse;
    float *pm, *pl, *zl;                         // E_LSE: (slices, Rp) maxima and sums, label logits
    op16* dz; long dz_plane; int dz_ld;          // E_DZ
    void* out; long ldo; int accumulate;         // E_OUT: elements of elt; E_PART: fp32 (slice, m, n)
    long slice;
    int R, V, v0, Rp, label_bytes, operands;     // operands: 1 = dz and W (dx), 2 = x and dz (dW)
};
__device__ __forceinline__ long label_of(const Epi& e, int r) {
    return e.label_bytes == 8 ? (long)reinterpret_cast<const long long*>(e.labels)[r] : (long)reinterpret_cast<const int*>(e.labels)[r];
}

// C = A B^T over k, four waves as 2 x 2, each MT x NT tiles of 32 x 32
template <int MT, int NT, bool ADOWN, bool BDOWN, int EPI> __global__ __launch_bounds__(256) void product_kernel(Side A, Side B, Epi e, int mtiles, int ntiles, int ksteps, int slices) {
    constexpr int BM = 64 * MT, BN = 64 * NT, SA = BM * BK * 2, SB = BN * BK * 2;
    __shared__ __attribute__((aligned(16))) char lds[2][SA + SB];
    const int item = attn::xcd_item(mtiles * ntiles * slices);
    if (item < 0) return;
    const int nt = item % ntiles, mt = item / ntiles % mtiles, sl = item / ntiles / mtiles;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, wm = w >> 1, wn = w & 1, h = lane >> 5;
    const int m0 = mt * BM, n0 = nt * BN;
    const int per = (ksteps + slices - 1) / slices, k_lo = min(sl * per, ksteps), k_hi = min(k_lo + per, ksteps), steps = (k_hi - k_lo) * PAIRS;
    f32x16 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int x = 0; x < 16; ++x) acc[i][j][x] = 0.f;
    Loader<BM, ADOWN> la;
    Loader<BN, BDOWN> lb;
    // fp32: the small products first (lo hi, hi lo), then hi hi, of one k step after the other
    const auto load = [&](int s) {
        const int k = (k_lo + s / PAIRS) * BK, p = s % PAIRS;
        la.load(A, A.p + (PAIRS == 3 && p == 0 ? A.plane : 0), m0, k);
        lb.load(B, B.p + (PAIRS == 3 && p == 1 ? B.plane : 0), n0, k);
    };
    if (steps) load(0);
    for (int s = 0; s < steps; ++s) {
        char* t = lds[s & 1];
        la.store(t); lb.store(t + SA);
        __syncthreads();
        if (s + 1 < steps) load(s + 1);
#pragma unroll
        for (int q = 0; q < BK / 16; ++q) {
            u32x4 a[MT], b[NT];
#pragma unroll
            for (int i = 0; i < MT; ++i) a[i] = fragment<BM, ADOWN>(t, (wm * MT + i) * 32, q, lane);
#pragma unroll
            for (int j = 0; j < NT; ++j) b[j] = fragment<BN, BDOWN>(t + SA, (wn * NT + j) * 32, q, lane);
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int j = 0; j < NT; ++j) acc[i][j] = attn::mma<op16>(a[i], b[j], acc[i][j]);
        }
    }
    const int mw = m0 + wm * MT * 32, nw = n0 + wn * NT * 32;
    if constexpr (EPI == E_LSE || EPI == E_DZ) {                  // m: vocabulary entries (from v0 on), n: rows of x
        float f = 1.f, gs = 1.f;
        if constexpr (NPL == 2) f = ldexpf(1.f, -up_exp(max_of(e.part_x)) - up_exp(max_of(e.part_w)));
        if constexpr (EPI == E_DZ) gs = ldexpf(1.f, DZ_BITS - g_exp(max_of(e.part_g)));
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            const int r = nw + 32 * j + (lane & 31);
            const long lab = r < e.R ? label_of(e, r) : -1;
            if constexpr (EPI == E_LSE) {
                float top = -INFINITY;
#pragma unroll
                for (int i = 0; i < MT; ++i)
#pragma unroll
                    for (int x = 0; x < 16; ++x) {
                        const int v = mw + 32 * i + 8 * (x >> 2) + 4 * h + (x & 3);
                        float z = acc[i][j][x] * f;
                        if (e.bias) z += v < e.V ? (float)e.bias[v] : 0.f;
                        if (v == lab && v < e.V) e.zl[r] = z;
                        z = v < e.V ? z : -INFINITY;
                        acc[i][j][x] = z;
                        top = fmaxf(top, z);
                    }
                top = attn::half_max(top);
                const float base = top == -INFINITY ? 0.f : top;
                float l = 0.f;
#pragma unroll
                for (int i = 0; i < MT; ++i)
#pragma unroll
                    for (int x = 0; x < 16; ++x) l += __builtin_amdgcn_exp2f((acc[i][j][x] - base) * LOG2E);
                l = attn::half_sum(l);
                if (h == 0 && r < e.Rp) { const long at = (long)(mt * 2 + wm) * e.Rp + r; e.pm[at] = top; e.pl[at] = l; }
            } else {
                const bool has = lab >= 0 && lab < e.V;
                const float g = has ? e.dloss[min(r, e.R - 1)] * gs : 0.f, lse = has ? e.lse[min(r, e.R - 1)] : INFINITY;
                if (r >= e.Rp) continue;
#pragma unroll
                for (int i = 0; i < MT; ++i)
#pragma unroll
                    for (int a = 0; a < 4; ++a) {
                        const int c = mw + 32 * i + 8 * a + 4 * h;              // column of the piece
                        if (c >= e.dz_ld) continue;
                        typename Num<op16>::x4 hi, lo;
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            const int v = e.v0 + c + x;
                            float z = acc[i][j][4 * a + x] * f;
                            if (e.bias) z += v < e.V ? (float)e.bias[v] : 0.f;
                            float d = has && v < e.V ? g * (__builtin_amdgcn_exp2f((z - lse) * LOG2E) - (v == lab ? 1.f : 0.f)) : 0.f;
                            hi[x] = (op16)d;
                            lo[x] = (op16)(d - (float)hi[x]);
                        }
                        *reinterpret_cast<typename Num<op16>::x4*>(e.dz + (long)r * e.dz_ld + c) = hi;
                        if constexpr (NPL == 2) *reinterpret_cast<typename Num<op16>::x4*>(e.dz + e.dz_plane + (long)r * e.dz_ld + c) = lo;
                    }
            }
        }
    } else {
        int ex = g_exp(max_of(e.part_g)) - DZ_BITS;
        if constexpr (NPL == 2) ex -= up_exp(max_of(e.operands == 1 ? e.part_w : e.part_x));
        const float f = ldexpf(1.f, ex);
        const int N = e.V;                                        // (the columns that exist)
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            const int n = nw + 32 * j + (lane & 31);
            if (n >= N) continue;
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int x = 0; x < 16; ++x) {
                    const int m = mw + 32 * i + 8 * (x >> 2) + 4 * h + (x & 3);
                    if (m >= e.R) continue;                       // (R: the rows that exist)
                    const float v = acc[i][j][x] * f;
                    if constexpr (EPI == E_OUT) {
                        elt* o = reinterpret_cast<elt*>(e.out) + m * e.ldo + n;
                        *o = (elt)(e.accumulate ? (float)*o + v : v);
                    } else {
                        float* o = reinterpret_cast<float*>(e.out) + sl * e.slice + m * e.ldo + n;
                        *o = e.accumulate ? *o + v : v;
                    }
                }
        }
    }
}

// lse and loss of a row from its slices' maxima and sums: 32 rows x 8 lanes a block
__global__ __launch_bounds__(256) void finish_kernel(const float* __restrict__ pm, const float* __restrict__ pl, const float* __restrict__ zl, const void* __restrict__ labels, int label_bytes,
                                                     float* __restrict__ loss, float* __restrict__ lse, int R, int Rp, int V, int slices) {
    __shared__ float sm[8][32], ss[8][32];
    const int c = threadIdx.x & 31, g = threadIdx.x >> 5, r = blockIdx.x * 32 + c;
    float m = -INFINITY, l = 0.f;
    if (r < R) {
        for (int s = g; s < slices; s += 8) m = fmaxf(m, pm[(long)s * Rp + r]);
        for (int s = g; s < slices; s += 8) {
            const float a = pm[(long)s * Rp + r];
            l += pl[(long)s * Rp + r] * (a == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((a - m) * LOG2E));
        }
    }
    sm[g][c] = m; ss[g][c] = l;
    __syncthreads();
    if (g || r >= R) return;
    float M = m;
#pragma unroll
    for (int x = 1; x < 8; ++x) M = fmaxf(M, sm[x][c]);
    float L = 0.f;
#pragma unroll
    for (int x = 0; x < 8; ++x) L += ss[x][c] * (sm[x][c] == -INFINITY ? (ss[x][c] == 0.f ? 0.f : 1.f) : __builtin_amdgcn_exp2f((sm[x][c] - M) * LOG2E));
    const float s = M + logf(L);
    const long lab = label_bytes == 8 ? (long)reinterpret_cast<const long long*>(labels)[r] : (long)reinterpret_cast<const int*>(labels)[r];
    if (lse) lse[r] = s;
    if (loss) loss[r] = lab >= 0 && lab < V ? s - zl[r] : 0.f;
}

// out (rows, cols) (+)= sum of the slices
__global__ __launch_bounds__(256) void sum_slices_kernel(const float* __restrict__ part, int slices, long slice, long rows, int cols, long ldp, elt* __restrict__ out, long ldo, int accumulate) {
    const long n = rows * cols;
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long)gridDim.x * 256) {
        const long r = i / cols, c = i - r * cols;
        float v = 0.f;
        for (int s = 0; s < slices; ++s) v += part[s * slice + r * ldp + c];
        elt* o = out + r * ldo + c;
        *o = (elt)(accumulate ? (float)*o + v : v);
    }
}

// db: column sums of a dz piece, 256 rows a block -> partial sums (slices, cols); joined by sum_slices_kernel
constexpr int DB_ROWS = 256;
__global__ __launch_bounds__(256) void colsum_kernel(const op16* __restrict__ dz, long plane, int ld, int rows, const float* __restrict__ part_g, float* __restrict__ part) {
    __shared__ float red[32][65];
    const int ch = threadIdx.x & 7, g = threadIdx.x >> 3, c = blockIdx.x * 64 + ch * 8;
    float s[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) s[k] = 0.f;
    if (c < ld)
        for (int r = blockIdx.y * DB_ROWS + g; r < min((int)(blockIdx.y + 1) * DB_ROWS, rows); r += 32)
#pragma unroll
            for (int p = NPL - 1; p >= 0; --p) {
                const auto v = *reinterpret_cast<const typename Num<op16>::x16*>(dz + p * plane + (long)r * ld + c);
#pragma unroll
                for (int k = 0; k < 8; ++k) s[k] += (float)v[k];
            }
#pragma unroll
    for (int k = 0; k < 8; ++k) red[g][ch * 8 + k] = s[k];
    __syncthreads();
    const float f = ldexpf(1.f, g_exp(max_of(part_g)) - DZ_BITS);
    if (threadIdx.x < 64 && blockIdx.x * 64 + threadIdx.x < ld) {
        float v = 0.f;
#pragma unroll
        for (int k = 0; k < 32; ++k) v += red[k][threadIdx.x];
        part[(long)blockIdx.y * ld + blockIdx.x * 64 + threadIdx.x] = v * f;
    }
}

// ---- plan of a call: what is packed, the pieces, the workspace
struct Plan {
    int Rp, Dp, Vp;                     // rows, hidden width and vocabulary rounded up to the contraction step
    bool pack_x, pack_w;
    int piece, pieces;
    int dx_slices, dw_slices, db_slices, lse_slices;
    bool dx_parts;
    size_t parts, xo, wo, a, b, zl, dz, dxp, dwp, dbp, bytes;      // offsets
};
static size_t up(size_t n) { return (n + 255) & ~(size_t)255; }
static int up32(int n) { return (n + 31) & ~31; }
static int cut(long tiles, int ksteps) {                          // slices of a contraction whose tiles alone do not fill the chip
    if (tiles >= 192) return 1;
    const long s = 384 / tiles, most = ksteps / 8;                // eight steps a slice at least
    return (int)(s < 1 || most < 1 ? 1 : s < most ? s : most);
}

static bool bad(const sarVocabCe* a) {
    return !a || a->R < 1 || a->D < 1 || a->V < 1 || a->R > (1 << 24) || a->D > (1 << 16) || a->V > (1 << 24) || (a->label_bytes != 4 && a->label_bytes != 8) || a->ldx < a->D || a->ldk < a->V ||
           (a->R + 127L) / 128 * ((a->V + 127L) / 128) > (1L << 28);
}
static Plan plan(const sarVocabCe* a, bool grad) {
    Plan p = {};
    p.Rp = up32(a->R); p.Dp = up32(a->D); p.Vp = up32(a->V);
    // operands are read where they lie when their rows are 16-byte aligned and no row ends inside a contraction step; fp32 ones become planes
    p.pack_x = NPL == 2 || a->D % 32 || a->ldx % 8 || (uintptr_t)a->x % 16;
    p.pack_w = NPL == 2 || a->V % 32 || a->ldk % 8 || (uintptr_t)a->kernel % 16;
    size_t at = 0;
    const auto take = [&](size_t n) { const size_t o = at; at += up(n); return o; };
    p.parts = take(3 * PARTS * 4);
    if (p.pack_x) p.xo = take((size_t)a->R * p.Dp * 2 * NPL);
    if (p.pack_w) p.wo = take((size_t)a->D * p.Vp * 2 * NPL);
    p.lse_slices = 2 * cdiv(a->V, 128);
    if (!grad) {
        p.a = take((size_t)p.lse_slices * p.Rp * 4); p.b = take((size_t)p.lse_slices * p.Rp * 4);
        p.zl = take((size_t)p.Rp * 4);
    } else {
        // a piece's dz: about 128 MB, which the 256 MB last-level cache holds between its writer and its two readers
        long w = (128L << 20) / ((long)p.Rp * 2 * NPL) / 256 * 256;
        if (w < 256) w = 256;
        p.pieces = cdiv(a->V, w);
        p.piece = (int)(p.pieces == 1 ? p.Vp : cdiv(cdiv(a->V, p.pieces), 256) * 256L);
        p.pieces = cdiv(a->V, p.piece);
        const int cols = p.piece < p.Vp ? p.piece : p.Vp;
        p.dx_slices = cut((long)cdiv(a->R, 128) * cdiv(a->D, 128), cols / 32);
        p.dw_slices = cut((long)cdiv(a->D, 128) * cdiv(cols, 128), p.Rp / 32);
        p.db_slices = cdiv(p.Rp, DB_ROWS);
        p.dx_parts = p.dx_slices > 1 || p.pieces > 1;
        p.dz = take((size_t)p.Rp * cols * 2 * NPL);
        if (p.dx_parts) p.dxp = take((size_t)p.dx_slices * a->R * a->D * 4);
        if (p.dw_slices > 1) p.dwp = take((size_t)p.dw_slices * a->D * cols * 4);
        if (a->dbias) p.dbp = take((size_t)p.db_slices * cols * 4);
    }
    p.bytes = at;
    return p;
}

template <typename T> static void absmax(const T* x, long rows, int cols, long ld, float* part, hipStream_t st) {
    hipLaunchKernelGGL((absmax_kernel<T>), dim3((unsigned)(rows < PARTS ? rows : PARTS)), dim3(256), 0, st, x, rows, cols, ld, part);
}
// the operands as the products read them
static void operands(const sarVocabCe* a, const Plan& p, Side& x, Side& w, hipStream_t st) {
    char* ws = reinterpret_cast<char*>(a->ws);
    float* parts = reinterpret_cast<float*>(ws + p.parts);
    x = {reinterpret_cast<const op16*>(a->x), 0, a->ldx, 0, 0};
    w = {reinterpret_cast<const op16*>(a->kernel), 0, a->ldk, 0, 0};
    if (p.pack_x) {
        x = {reinterpret_cast<op16*>(ws + p.xo), (long)a->R * p.Dp, p.Dp, 0, 0};
        if (NPL == 2) absmax(reinterpret_cast<const elt*>(a->x), a->R, a->D, a->ldx, parts, st);
        const long n = (long)a->R * p.Dp / 8;
        hipLaunchKernelGGL((pack_kernel<elt>), dim3((unsigned)(n < 2048 * 256 ? (n + 255) / 256 : 2048)), dim3(256), 0, st, reinterpret_cast<const elt*>(a->x), a->R, a->D, a->ldx, const_cast<op16*>(x.p), x.plane, p.Dp, parts);
    }
    if (p.pack_w) {
        w = {reinterpret_cast<op16*>(ws + p.wo), (long)a->D * p.Vp, p.Vp, 0, 0};
        if (NPL == 2) absmax(reinterpret_cast<const elt*>(a->kernel), a->D, a->V, a->ldk, parts + PARTS, st);
        const long n = (long)a->D * p.Vp / 8;
        hipLaunchKernelGGL((pack_kernel<elt>), dim3((unsigned)(n < 2048 * 256 ? (n + 255) / 256 : 2048)), dim3(256), 0, st, reinterpret_cast<const elt*>(a->kernel), a->D, a->V, a->ldk, const_cast<op16*>(w.p), w.plane, p.Vp, parts + PARTS);
    }
}
template <int MT, int NT, bool AD, bool BD, int EPI> static void product(Side A, Side B, const Epi& e, int m, int n, int ksteps, int slices, hipStream_t st) {
    const int mt = cdiv(m, 64 * MT), nt = cdiv(n, 64 * NT);
    hipLaunchKernelGGL((product_kernel<MT, NT, AD, BD, EPI>), dim3((unsigned)attn::xcd_grid((long)mt * nt * slices)), dim3(256), 0, st, A, B, e, mt, nt, ksteps, slices);
}

}
using namespace SAR_FN(vce);

extern "C" size_t SAR_WS(sar_vocab_ce_fwd)(const sarVocabCe* a) { return bad(a) ? 0 : plan(a, false).bytes; }
extern "C" size_t SAR_WS(sar_vocab_ce_bwd)(const sarVocabCe* a) { return bad(a) ? 0 : plan(a, true).bytes; }

extern "C" int SAR_FN(sar_vocab_ce_fwd)(const sarVocabCe* a, hipStream_t st) {
    if (bad(a) || !a->x || !a->kernel || !a->labels || (!a->loss && !a->lse) || !a->ws || (uintptr_t)a->ws % 256) return SAR_EINVAL;
    const Plan p = plan(a, false);
    if (a->ws_bytes < 0 || (size_t)a->ws_bytes < p.bytes) return SAR_EINVAL;
    char* ws = reinterpret_cast<char*>(a->ws);
    float* parts = reinterpret_cast<float*>(ws + p.parts);
    Side x, w;
    operands(a, p, x, w, st);
    w.len = p.pack_w ? p.Vp : a->V; w.k = a->D;
    x.len = a->R; x.k = p.Dp;
    Epi e = {};
    e.part_x = parts; e.part_w = parts + PARTS;
    e.bias = reinterpret_cast<const elt*>(a->bias); e.labels = a->labels; e.label_bytes = a->label_bytes;
    e.pm = reinterpret_cast<float*>(ws + p.a); e.pl = reinterpret_cast<float*>(ws + p.b); e.zl = reinterpret_cast<float*>(ws + p.zl);
    e.R = a->R; e.V = a->V; e.Rp = p.Rp;
    product<2, 2, true, false, E_LSE>(w, x, e, a->V, a->R, p.Dp / BK, 1, st);
    hipLaunchKernelGGL(finish_kernel, dim3((unsigned)cdiv(a->R, 32)), dim3(256), 0, st, e.pm, e.pl, e.zl, a->labels, a->label_bytes, a->loss, a->lse, a->R, p.Rp, a->V, p.lse_slices);
    SAR_CHECK_LAUNCH();
    return SAR_OK;
}

extern "C" int SAR_FN(sar_vocab_ce_bwd)(const sarVocabCe* a, hipStream_t st) {
    if (bad(a) || !a->x || !a->kernel || !a->labels || !a->dloss || !a->lse || !a->ws || (uintptr_t)a->ws % 256 || (!a->dx && !a->dkernel && !a->dbias) || (a->accumulate && SAR_ELT != 0)) return SAR_EINVAL;
    const Plan p = plan(a, true);
    if (a->ws_bytes < 0 || (size_t)a->ws_bytes < p.bytes) return SAR_EINVAL;
    char* ws = reinterpret_cast<char*>(a->ws);
    float* parts = reinterpret_cast<float*>(ws + p.parts);
    op16* dz = reinterpret_cast<op16*>(ws + p.dz);
    Side x, w;
    operands(a, p, x, w, st);
    absmax(a->dloss, 1, a->R, a->R, parts + 2 * PARTS, st);
    for (int i = 0; i < p.pieces; ++i) {
        const int v0 = i * p.piece, cols = a->V - v0 < p.piece ? a->V - v0 : p.piece, ld = up32(cols);
        const long plane = (long)p.Rp * ld;
        Epi e = {};
        e.part_x = parts; e.part_w = parts + PARTS; e.part_g = parts + 2 * PARTS;
        e.bias = reinterpret_cast<const elt*>(a->bias); e.labels = a->labels; e.label_bytes = a->label_bytes; e.dloss = a->dloss; e.lse = a->lse;
        e.dz = dz; e.dz_plane = plane; e.dz_ld = ld;
        e.R = a->R; e.V = a->V; e.v0 = v0; e.Rp = p.Rp;
        Side ws_ = w, xs = x;
        ws_.p += v0; ws_.len = (p.pack_w ? p.Vp : a->V) - v0; ws_.k = a->D;
        xs.len = a->R; xs.k = p.Dp;
        product<2, 2, true, false, E_DZ>(ws_, xs, e, ld, p.Rp, p.Dp / BK, 1, st);
        if (a->dx) {
            Epi o = e;
            o.R = a->R; o.V = a->D; o.operands = 1; o.ldo = a->D;
            Side A = {dz, plane, ld, p.Rp, ld}, B = {w.p + v0, w.plane, w.ld, a->D, ld};
            if (p.dx_parts) {
                o.out = ws + p.dxp; o.slice = (long)a->R * a->D; o.accumulate = i > 0;
                product<2, 2, false, false, E_PART>(A, B, o, a->R, a->D, ld / BK, p.dx_slices, st);
            } else {
                o.out = a->dx; o.accumulate = 0;
                product<2, 2, false, false, E_OUT>(A, B, o, a->R, a->D, ld / BK, 1, st);
            }
        }
        if (a->dkernel) {
            Epi o = e;
            o.R = a->D; o.V = cols; o.operands = 2;
            Side A = {x.p, x.plane, x.ld, p.pack_x ? p.Dp : a->D, a->R}, B = {dz, plane, ld, ld, p.Rp};
            elt* out = reinterpret_cast<elt*>(a->dkernel) + v0;
            if (p.dw_slices > 1) {
                o.out = ws + p.dwp; o.slice = (long)a->D * ld; o.ldo = ld; o.accumulate = 0;
                product<2, 2, true, true, E_PART>(A, B, o, a->D, cols, p.Rp / BK, p.dw_slices, st);
                const long n = (long)a->D * cols;
                hipLaunchKernelGGL(sum_slices_kernel, dim3((unsigned)(n < 4096 * 256 ? (n + 255) / 256 : 4096)), dim3(256), 0, st, reinterpret_cast<float*>(ws + p.dwp), p.dw_slices, o.slice, (long)a->D, cols, (long)ld, out, (long)a->V, a->accumulate);
            } else {
                o.out = out; o.ldo = a->V; o.accumulate = a->accumulate;
                product<2, 2, true, true, E_OUT>(A, B, o, a->D, cols, p.Rp / BK, 1, st);
            }
        }
        if (a->dbias) {
            float* part = reinterpret_cast<float*>(ws + p.dbp);
            hipLaunchKernelGGL(colsum_kernel, dim3((unsigned)cdiv(ld, 64), (unsigned)p.db_slices), dim3(256), 0, st, dz, plane, ld, p.Rp, parts + 2 * PARTS, part);
            hipLaunchKernelGGL(sum_slices_kernel, dim3((unsigned)cdiv(cols, 256)), dim3(256), 0, st, part, p.db_slices, (long)ld, 1L, cols, (long)ld, reinterpret_cast<elt*>(a->dbias) + v0, (long)cols, a->accumulate);
        }
    }
    if (a->dx && p.dx_parts) {
        const long n = (long)a->R * a->D;
        hipLaunchKernelGGL(sum_slices_kernel, dim3((unsigned)(n < 4096 * 256 ? (n + 255) / 256 : 4096)), dim3(256), 0, st, reinterpret_cast<float*>(ws + p.dxp), p.dx_slices, n, (long)a->R, a->D, (long)a->D, reinterpret_cast<elt*>(a->dx), (long)a->D, 0);
    }
    SAR_CHECK_LAUNCH();
    return SAR_OK;
}
