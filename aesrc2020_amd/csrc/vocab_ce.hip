// Softmax cross entropy over a vocabulary straight from the hidden rows and the output layer's (D, V) kernel, without a (R, V) array of
// logits or probabilities.
//
//   z = x W + b    lse_r = log sum_v exp z_rv    loss_r = lse_r - z_{r, label}    (0 for a label outside [0, V))
//   dz_rv = g_r (exp(z_rv - lse_r) - [v = label_r])    dx = dz W^T    dW = x^T dz    db = sum_r dz
//
// Forward: one product whose epilogue keeps the maximum and the sum of every 128 (64) vocabulary entries of a row; a small kernel joins them.
// Backward, in pieces of the vocabulary: the piece's logits are computed again, turned into dz in the epilogue and written once in the
// operand type; two more products read that piece (it stays in the last-level cache) for dx and dW.
//
// The products run on the 32x32x16 matrix instructions (small fp32 ones on the fp32 ones: direct()).
// fp32 operands are two fp16 planes under a power of two that puts the largest element in [2^13, 2^14): hi + lo hold 22 bits of elements down to 2^-16
// of that one (below, 2^-38 of it), hi hi + hi lo + lo hi is the product to 2^-22 or so of |a| |b|, at a third of the fp16 rate (the fp32 matrix
// instructions run at a sixteenth).  For the logits every row of x has its own scale, so that no row reaches another's results; W has one.
// dz is held in fp16, times 2^14 and a power of two that puts |g| into [1/2, 1): every probability down to 2^-28 is a normal number with 11 bits.  For bf16
// the backward therefore takes x and W in fp16 too (their 8 bits are exact down to 2^-31 of the largest), which leaves the gradients the accuracy of
// their own rounding.  Where operands are packed (fp32, bf16) that power is each row's own, which dx takes back by row.  dW = x^T dz sums over the rows, so
// there x is packed a second time, times the rows' powers, under one scale; rows without a label are zeros.  An element of dW is good to 2^-38 of the
// largest |x g|.  fp16 x lies where it is, and g's power is one for all rows with a label.
// Compiled once per element type: SAR_ELT 0 = fp32, 1 = bf16, 2 = fp16.
#include "attn_tiles.h"

#if SAR_ELT == 0
typedef float elt;
typedef _Float16 fwd16;                 // operand type of the forward's product, and of the backward's three
typedef _Float16 bwd16;
#define SAR_FN(n) n##_f32
#define SAR_WS(n) n##_f32_workspace_bytes
#elif SAR_ELT == 1
typedef __bf16 elt;
typedef __bf16 fwd16;
typedef _Float16 bwd16;
#define SAR_FN(n) n##_bf16
#define SAR_WS(n) n##_bf16_workspace_bytes
#else
typedef _Float16 elt;
typedef _Float16 fwd16;
typedef _Float16 bwd16;
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
template <int PITCH> __device__ __forceinline__ int chunk_at(int row, int ch) { return attn::chunk_at<PITCH, true>(row, ch); }
using attn::as16;

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr int NPL = SAR_ELT == 0 ? 2 : 1;
constexpr bool FWD_SCALED = SAR_ELT == 0, BWD_SCALED = SAR_ELT != 2;           // operands packed under powers of two
constexpr int DZ_BITS = 14;

// Device scalars of a call: maxima of |x| (rows with a label), |W| and |dloss| (the same rows), reduced from 256 partial maxima each by whoever reads them
constexpr int PARTS = 256;
enum { PART_X, PART_W, PART_G };
__device__ __forceinline__ float max_of(const float* part) {
    const int l = threadIdx.x & 63;
    return wave_max(fmaxf(fmaxf(part[l], part[l + 64]), fmaxf(part[l + 128], part[l + 192])));
}
// Scales are exponents, applied by ldexp: 2^e itself may leave fp32's range where the product with it does not.
__device__ __forceinline__ float times2(float v, int e) { return __builtin_amdgcn_ldexpf(v, e); }
__device__ __forceinline__ int g_exp(float v) {                   // v 2^-e in [1/2, 1) (0 for v = 0)
    int e = 0;
    (void)frexpf(v, &e);
    return v == 0.f ? 0 : e;
}
__device__ __forceinline__ int up_exp(float v) { return v == 0.f ? 0 : DZ_BITS - g_exp(v); }      // v 2^e in [2^13, 2^14)

// labels (R) of 4 or 8 bytes; a row whose label lies outside [0, V) is left out
struct Labels { const void* p; int bytes, V; };
__device__ __forceinline__ long label_of(const Labels& l, long r) {
    return l.bytes == 8 ? (long)reinterpret_cast<const long long*>(l.p)[r] : (long)reinterpret_cast<const int*>(l.p)[r];
}
__device__ __forceinline__ bool counts(const Labels& l, long r) {
    const long v = label_of(l, r);
    return v >= 0 && v < l.V;
}

enum { MAX_ALL, MAX_ROWS, MAX_G };       // of a whole tensor, of its rows with a label times their g's powers of two, of dloss
struct MaxJob { const void* x; long rows, ld; int cols, kind, part; };
struct MaxJobs { MaxJob j[3]; Labels labels; const float* dloss; };
// partial maxima of the finite |values| of up to three tensors (blockIdx.y): PARTS places each.  What a row that is left out holds must not decide how
// finely the others' x and dz are held.
__global__ __launch_bounds__(1024) void absmax_kernel(MaxJobs jobs, float* __restrict__ part) {
    __shared__ float red[16];
    const MaxJob j = jobs.j[blockIdx.y];
    constexpr int V = Num<elt>::PER;
    float m = 0.f;
    const auto see = [&](float v) { v = fabsf(v); if (v < INFINITY) m = fmaxf(m, v); };
    // n elements at p, by threads `first`, first + step, ...: sixteen bytes each where p and n allow it
    const auto row = [&](const elt* p, long n, bool wide, long first, long step) {
        if (wide) {
            const auto* q = reinterpret_cast<const typename Num<elt>::x16*>(p);
            long c = first;
            n /= V;
            for (; c + 3 * step < n; c += 4 * step) {             // four loads in flight
                const auto a = q[c], b = q[c + step], d = q[c + 2 * step], e = q[c + 3 * step];
#pragma unroll
                for (int k = 0; k < V; ++k) { see((float)a[k]); see((float)b[k]); see((float)d[k]); see((float)e[k]); }
            }
            for (; c < n; c += step) {
                const auto a = q[c];
#pragma unroll
                for (int k = 0; k < V; ++k) see((float)a[k]);
            }
        } else
            for (long c = first; c < n; c += step) see((float)p[c]);
    };
    const elt* x = reinterpret_cast<const elt*>(j.x);
    const bool aligned = (uintptr_t)j.x % 16 == 0, wide = aligned && j.cols % V == 0 && j.ld % V == 0;
    if (j.kind == MAX_G) {
        for (long c = blockIdx.x * 1024 + threadIdx.x; c < j.cols; c += PARTS * 1024)
            if (counts(jobs.labels, c)) see(reinterpret_cast<const float*>(j.x)[c]);
    } else if (j.kind == MAX_ROWS) {                              // a wave per row
        for (long r = blockIdx.x * 16 + (threadIdx.x >> 6); r < j.rows; r += PARTS * 16)
            if (counts(jobs.labels, r)) {
                const float before = m;
                m = 0.f;
                row(x + r * j.ld, j.cols, wide, threadIdx.x & 63, 64);
                const float here = times2(m, g_exp(jobs.dloss[r]));
                m = before;
                see(here);
            }
    } else if (j.ld == j.cols) {                                  // no gaps: as one row
        row(x, j.rows * j.cols, aligned && j.rows * j.cols % V == 0, (long)blockIdx.x * 1024 + threadIdx.x, PARTS * 1024);
    } else {
        for (long r = blockIdx.x; r < j.rows; r += PARTS) row(x + r * j.ld, j.cols, wide, threadIdx.x, 1024);
    }
    m = block_max(m, red);
    if (threadIdx.x == 0) part[j.part * PARTS + blockIdx.x] = m;
}

// rows of `cols` elements -> rows of `pitch` operand elements, zeros behind (SCALED: planes hi, lo of fp32), for x and W (blockIdx.y).  The scale comes from
// `part`'s maxima; or, with row_e, every row has its own, whose exponent is left there (row_e[r]; g's in row_e[row_places(rows) + r] if there is a dloss), and with `all`
// the rows go there too, times g's power and under the scale of `part`, those without a label as zeros.
// exponents of rows: so many places, that a tile's rows have one each (what those behind the last row hold meets zeros only)
__device__ __host__ __forceinline__ int row_places(int rows) { return (rows + 63) / 64 * 64 + 64; }
struct PackJob { const elt* x; void* y; long rows, ld, plane; int cols, pitch; const float* part; int* row_e; void* all; };
struct PackJobs { PackJob j[2]; Labels labels; const float* dloss; };
template <typename OP, bool SCALED> __global__ __launch_bounds__(256) void pack_kernel(PackJobs jobs) {
    const PackJob j = jobs.j[blockIdx.y];
    const auto fetch = [&](long r, int c, elt (&v)[8]) {
        const elt* p = j.x + r * j.ld + c;
        if (c + 8 <= j.cols) {
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = p[k];
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = c + k < j.cols ? p[k] : (elt)0.f;
        }
    };
    const auto put = [&](void* to, long r, int c, const elt (&v)[8], int e, bool none) {
        constexpr int PER = Num<OP>::PER;
        OP* y = reinterpret_cast<OP*>(to) + r * j.pitch + c;
        typename Num<OP>::x16 hi[8 / PER], lo[8 / PER];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const float s = none ? 0.f : SCALED ? times2((float)v[k], e) : (float)v[k];
            hi[k / PER][k % PER] = (OP)s;
            if constexpr (SCALED && NPL == 2) lo[k / PER][k % PER] = (OP)(s - (float)hi[k / PER][k % PER]);
        }
#pragma unroll
        for (int q = 0; q < 8 / PER; ++q) {
            *reinterpret_cast<typename Num<OP>::x16*>(y + q * PER) = hi[q];
            if constexpr (SCALED && NPL == 2) *reinterpret_cast<typename Num<OP>::x16*>(y + j.plane + q * PER) = lo[q];
        }
    };
    const int all = SCALED && j.part ? up_exp(max_of(j.part)) : 0;
    elt v[8];
    if (SCALED && j.row_e) {                                      // a wave per row, which it reads twice if it is wider than 512
        const int lane = threadIdx.x & 63;
        for (long r = (long)blockIdx.x * 4 + (threadIdx.x >> 6); r < j.rows; r += (long)gridDim.x * 4) {
            float m = 0.f;
            const bool in = jobs.dloss && counts(jobs.labels, r);
            const int eg = in ? g_exp(jobs.dloss[r]) : 0;
            for (int c = lane * 8; c < j.pitch; c += 512) {
                fetch(r, c, v);
#pragma unroll
                for (int k = 0; k < 8; ++k) { const float a = fabsf((float)v[k]); if (a < INFINITY) m = fmaxf(m, a); }
            }
            const int e = up_exp(wave_max(m));
            if (lane == 0) {
                j.row_e[r] = e;
                if (jobs.dloss) j.row_e[row_places((int)j.rows) + r] = eg;
            }
            for (int c = lane * 8; c < j.pitch; c += 512) {
                if (j.pitch > 512) fetch(r, c, v);
                put(j.y, r, c, v, e, false);
                if (j.all) put(j.all, r, c, v, all + eg, !in);
            }
        }
        return;
    }
    // a block takes 256 pieces of eight of one row, then the next block's
    const int across = (j.pitch / 8 + 255) / 256;
    for (long i = blockIdx.x; i < j.rows * across; i += gridDim.x) {
        const long r = i / across;
        const int c = ((int)(i - r * across) * 256 + threadIdx.x) * 8;
        if (c >= j.pitch) continue;
        fetch(r, c, v);
        put(j.y, r, c, v, all, false);
    }
}

// One operand of a product: `len` rows or columns (the output's side), contraction length k.
// DOWN = false: element (i, k) at p[i ld + k] (k contiguous).  DOWN = true: element (i, k) at p[k ld + i] (read down the columns).
struct Side { const void* p; long plane, ld; int len, k; };

// an operand's LDS tile of one stage: ROWS of the output's side, BK of the contraction; everything outside the tensor arrives as zeros
// TAIL: the contraction may end inside a step (64 x 64 tiles; the larger ones' loads are 3 % slower with it and take packed operands instead)
template <typename OP, int BK, int ROWS, bool DOWN, bool TAIL> struct Operand {
    static constexpr int E = sizeof(OP), P = DOWN ? ROWS * E : BK * E, LINES = DOWN ? BK : ROWS, N = attn::TileLoader<P, LINES, true>::N;
    attn::TileLoader<P, LINES, true> loader;
    unsigned tail;                               // the loader's offsets for the last, shorter step along the contraction
    const OP* base;
    long ld;
    int lines, last;
    unsigned useful;
    __device__ __forceinline__ Operand(const Side& s, int i0)
        : loader((unsigned)(s.ld * E), DOWN ? (unsigned)min(ROWS, s.len - i0) * E : BK * E), tail(attn::TileLoader<P, LINES, true>((unsigned)(s.ld * E), DOWN ? 0 : (unsigned)(s.k % BK) * E).first),
          base(reinterpret_cast<const OP*>(s.p) + (DOWN ? i0 : i0 * s.ld)), ld(s.ld), lines(DOWN ? s.k : s.len - i0), last(DOWN ? 1 << 30 : s.k - BK),
          useful(DOWN ? (unsigned)min(ROWS, s.len - i0) * E : BK * E) {}
    __device__ __forceinline__ void load(int k, long plane, char* to, int wave) {
        const OP* p = base + plane + (DOWN ? k * ld : k);
        if constexpr (TAIL && !DOWN) {
            if (k > last) loader.first = tail;                    // (what lies behind is the next row; k only grows)
            loader.load(p, k < last + BK ? lines : 0, (unsigned)(ld * E), k <= last ? useful : (unsigned)(last + BK - k) * E, to, wave);
        } else loader.load(p, DOWN ? lines - k : lines, (unsigned)(ld * E), useful, to, wave);
    }
    // operand fragment: 32 rows at i0, sixteen (fp32: eight) contraction elements from the s-th such group on
    static __device__ __forceinline__ u32x4 fragment(const char* tile, int i0, int s, int lane) {
        if constexpr (DOWN && E == 4) {
            const int i = i0 + (lane & 31), k = 8 * s + 4 * (lane >> 5);
            u32x4 v;
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = *reinterpret_cast<const unsigned*>(tile + chunk_at<P>(k + j, i >> 2) + (i & 3) * 4);
            return v;
        } else if constexpr (DOWN) {
            const int i = lane & 15, k = 16 * s + 8 * (lane >> 5) + (i >> 2), ch = (i0 >> 3) + 2 * ((lane >> 4) & 1) + ((i >> 1) & 1), off = (i & 1) * 8;
            const u32x2 a = attn::tr16(tile + chunk_at<P>(k, ch) + off), b = attn::tr16(tile + chunk_at<P>(k + 4, ch) + off);
            return u32x4{a[0], a[1], b[0], b[1]};
        } else return *reinterpret_cast<const u32x4*>(tile + chunk_at<P>(i0 + (lane & 31), 2 * s + (lane >> 5)));
    }
};

// where the scale of dz comes from: bf16 planes and fp32 need none; packed rows have their own; a few fp16 rows are looked through by every wave, more by a
// launch of their own
enum { G_ONE, G_EACH, G_ROWS, G_PARTS };
constexpr int G_FEW = 1024;
// what happens to a finished tile: C (m, n), column n = lane % 32 of a 32 x 32 tile
enum { E_LSE, E_DZ, E_GRAD };
struct Epi {
    const float* parts;                          // maxima: PART_X, PART_W, PART_G
    const int *row_e, *g_e;                      // packed operands: exponents of x's scales, and of dloss, a row each
    const elt* bias;
    Labels labels;
    const float *dloss, *lse;
    float *pm, *pl, *zl;                         // E_LSE: (m tiles, Rp) maxima and sums, label logits
    float *loss, *lse_out;                       // E_LSE, one m tile: the results themselves
    void* dz; long dz_plane; int dz_ld, g_from;  // E_DZ
    float* db;                                   // E_DZ: (n tiles, dz_ld) column sums, or NULL
    elt* db_out; int db_accumulate;              // E_DZ, one n tile: the sums themselves
    void* out; long ldo; int accumulate;         // E_GRAD: elements of elt, or, with `part`, fp32 (slice, m, n)
    long slice;
    int R, V, v0, Rp, R_all, part, with_w;       // with_w: dz W^T (dx), else x^T dz (dW)
};

// a row's results from its maximum, sum and label logit (all in powers of two)
__device__ __forceinline__ void finish_row(float* loss, float* lse, int r, float m, float l, float own, long lab, int V) {
    if (lse) lse[r] = (m + __builtin_amdgcn_logf(l)) * LN2;
    if (loss) loss[r] = lab >= 0 && lab < V ? (m - own + __builtin_amdgcn_logf(l)) * LN2 : 0.f;
}
__device__ __forceinline__ int dz_exp(const Epi& e, int r) { return DZ_BITS - e.g_e[r]; }      // G_EACH: dz is held times 2^this
__device__ __forceinline__ int dz_exp(const Epi& e) {             // the others'
    if (e.g_from == G_ONE) return 0;                              // (a bf16 has an fp32's range)
    if (e.g_from == G_PARTS) return DZ_BITS - g_exp(max_of(e.parts + PART_G * PARTS));
    float m = 0.f;
    for (int r = threadIdx.x & 63; r < e.R_all; r += 64) {
        const float v = fabsf(e.dloss[r]);
        if (counts(e.labels, r) && v < INFINITY) m = fmaxf(m, v);
    }
    return DZ_BITS - g_exp(wave_max(m));
}

struct Job { Side A, B; Epi e; int mtiles, ntiles, ksteps, slices; };
// a launch has fewer than 2^32 threads along an axis: blocks in rows of so many (a multiple of the XCDs; surplus blocks find no item)
constexpr unsigned LAUNCH_ROW = 1u << 22;
// C = A B^T over k, four waves as 2 x 2, each MT x NT tiles of 32 x 32.  ST stages of LDS, loads ST - 1 steps ahead.
// What bounds it (16 bits, 128 x 128 tiles): LDS hands out four 16-byte fragments for four matrix instructions of a wave and takes the stages' loads,
// about as many cycles as the matrix instructions need; with two blocks a CU those are busy 41 (dz) to 63 % (dW) of the time, at the 1.8 GHz that the
// power limit leaves: 0.82 (dz) to 1.07 PFLOP/s (dW) for an 8192 x 8192 piece against 1024.
// PA, PB: planes of the operands (1, or 2: hi, lo); PZ: planes of the dz that E_DZ writes
template <typename OP, int BK, int MT, int NT, bool AD, bool BD, int EPI, bool SCALED, int PA, int PB, int PZ> struct Product {
    static constexpr int BM = 64 * MT, BN = 64 * NT, SA = BM * BK * (int)sizeof(OP), SB = BN * BK * (int)sizeof(OP), STAGE = PA * SA + PB * SB,
                         ST = 49152 / STAGE < 4 ? (49152 / STAGE > 2 ? 49152 / STAGE : 2) : 4;
    static constexpr int LDS = ST * STAGE;
    static __device__ __forceinline__ void run(char* lds, int block, const Job& job);
};
template <typename OP, int BK, int MT, int NT, bool AD, bool BD, int EPI, bool SCALED, int PA, int PB, int PZ>
__global__ __launch_bounds__(256, (PA * PB == 1 && BK == 32 ? 3 : 2)) void product_kernel(Job job) {
    typedef Product<OP, BK, MT, NT, AD, BD, EPI, SCALED, PA, PB, PZ> P;
    __shared__ __attribute__((aligned(1024))) char lds[P::LDS];
    P::run(lds, blockIdx.x + LAUNCH_ROW * blockIdx.y, job);
}
// dW and dx of a piece in one launch, 64 x 64 tiles: neither fills the chip by itself
template <typename OP, int BKW, int BKX, bool SCALED, int PO, int PZ> __global__ __launch_bounds__(256, 2) void grads_kernel(Job dw, Job dx, int first) {
    typedef Product<OP, BKW, 1, 1, true, true, E_GRAD, SCALED, PO, PZ, PZ> W;
    typedef Product<OP, BKX, 1, 1, false, false, E_GRAD, SCALED, PZ, PO, PZ> X;
    __shared__ __attribute__((aligned(1024))) char lds[W::LDS > X::LDS ? W::LDS : X::LDS];
    if ((int)blockIdx.x < first) W::run(lds, blockIdx.x, dw);
    else X::run(lds, blockIdx.x - first, dx);
}
template <typename OP, int BK, int MT, int NT, bool AD, bool BD, int EPI, bool SCALED, int PA, int PB, int PZ>
__device__ __forceinline__ void Product<OP, BK, MT, NT, AD, BD, EPI, SCALED, PA, PB, PZ>::run(char* lds, int block, const Job& job) {
    const Side &A = job.A, &B = job.B;
    const Epi& e = job.e;
    const int mtiles = job.mtiles, ntiles = job.ntiles, ksteps = job.ksteps, slices = job.slices;
    typedef Operand<OP, BK, BM, AD, MT == 1> OA;
    typedef Operand<OP, BK, BN, BD, MT == 1> OB;
    constexpr int LOADS = PA * OA::N + PB * OB::N;
    const int item = attn::xcd_item(mtiles * ntiles * slices, block);
    if (item < 0) return;
    // eight m tiles by all n tiles, m fastest: the tiles in flight on an XCD share both operands in its L2
    const int sl = item / (mtiles * ntiles), tile = item - sl * mtiles * ntiles, band = tile / (8 * ntiles), high = min(8, mtiles - 8 * band);
    const int nt = (tile - band * 8 * ntiles) / high, mt = band * 8 + (tile - band * 8 * ntiles) % high;
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = w >> 1, wn = w & 1, h = lane >> 5;
    const int m0 = mt * BM, n0 = nt * BN;
    const int per = (ksteps + slices - 1) / slices, k_lo = min(sl * per, ksteps), steps = min(k_lo + per, ksteps) - k_lo;
    f32x16 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int x = 0; x < 16; ++x) acc[i][j][x] = 0.f;
    OA oa(A, m0);
    OB ob(B, n0);
    const auto load = [&](int s, char* to) {
        const int k = (k_lo + s) * BK;
#pragma unroll
        for (int p = 0; p < PA; ++p) oa.load(k, p * A.plane, to + p * SA, w);
#pragma unroll
        for (int p = 0; p < PB; ++p) ob.load(k, p * B.plane, to + PA * SA + p * SB, w);
    };
#pragma unroll
    for (int s = 0; s < ST - 1; ++s)
        if (s < steps) load(s, lds + s * STAGE);
    int cur = 0;
    for (int s = 0; s < steps; ++s) {
        if (s + ST - 1 <= steps) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((ST - 2) * LOADS) : "memory");
        else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        if (s + ST - 1 < steps) load(s + ST - 1, lds + (cur == 0 ? ST - 1 : cur - 1) * STAGE);
        const char *ta = lds + cur * STAGE, *tb = ta + PA * SA;
#pragma unroll
        for (int q = 0; q < BK * (int)sizeof(OP) / 32; ++q) {
            u32x4 a[PA][MT], b[PB][NT];
#pragma unroll
            for (int p = 0; p < PA; ++p)
#pragma unroll
                for (int i = 0; i < MT; ++i) a[p][i] = OA::fragment(ta + p * SA, (wm * MT + i) * 32, q, lane);
#pragma unroll
            for (int p = 0; p < PB; ++p)
#pragma unroll
                for (int j = 0; j < NT; ++j) b[p][j] = OB::fragment(tb + p * SB, (wn * NT + j) * 32, q, lane);
            // (waves in their products before waves that load: dW 140 -> 134 us, dx 160 -> 155 us for an 8192-wide piece; the logits do not mind)
            __builtin_amdgcn_s_setprio(1);
            // the small products first; lo lo is left out
#pragma unroll
            for (int c = 0; c < 3; ++c) {
                if (c == 0 ? PA < 2 : c == 1 ? PB < 2 : false) continue;
#pragma unroll
                for (int i = 0; i < MT; ++i)
#pragma unroll
                    for (int j = 0; j < NT; ++j) acc[i][j] = attn::mma<OP>(a[c == 0 ? PA - 1 : 0][i], b[c == 1 ? PB - 1 : 0][j], acc[i][j]);
            }
        }
        __builtin_amdgcn_s_setprio(0);
        cur = cur == ST - 1 ? 0 : cur + 1;
    }
    const int mw = wm * MT * 32, nw = wn * NT * 32;               // the wave's corner of the tile
    // logits in powers of two: y = (acc f + b) log2 e, entries behind the vocabulary -inf
    const auto logits = [&](int v0) {
        if constexpr (SCALED) {
            const int w_exp = up_exp(max_of(e.parts + PART_W * PARTS));
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                const int down = -w_exp - e.row_e[n0 + nw + 32 * j + (lane & 31)];
#pragma unroll
                for (int i = 0; i < MT; ++i)
#pragma unroll
                    for (int x = 0; x < 16; ++x) acc[i][j][x] = times2(acc[i][j][x], down);
            }
        }
        const int first = v0 + m0 + mw + 4 * h;
        if (v0 + m0 + BM <= e.V) {
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int a = 0; a < 4; ++a) {
                    float b[4] = {0.f, 0.f, 0.f, 0.f};
                    if (e.bias)
#pragma unroll
                        for (int x = 0; x < 4; ++x) b[x] = (float)e.bias[first + 32 * i + 8 * a + x] * LOG2E;
#pragma unroll
                    for (int j = 0; j < NT; ++j)
#pragma unroll
                        for (int x = 0; x < 4; ++x) acc[i][j][4 * a + x] = fmaf(acc[i][j][4 * a + x], LOG2E, b[x]);
                }
        } else {
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int x = 0; x < 16; ++x) {
                    const int v = first + 32 * i + 8 * (x >> 2) + (x & 3);
                    const float b = e.bias && v < e.V ? (float)e.bias[v] * LOG2E : 0.f;
#pragma unroll
                    for (int j = 0; j < NT; ++j) acc[i][j][x] = v < e.V ? fmaf(acc[i][j][x], LOG2E, b) : -INFINITY;
                }
        }
    };
    // f(i, x) for the place of entry `at` (of the wave's corner), if the lane holds it
    const auto place = [&](long at, auto&& f) {
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int x = 0; x < 16; ++x)
                if (at == 32 * i + 8 * (x >> 2) + 4 * h + (x & 3)) f(i, x);
    };
    if constexpr (EPI == E_LSE) {                                 // m: vocabulary entries, n: rows of x
        float* join = reinterpret_cast<float*>(lds);              // (3, BN): maxima, sums and label logits of the lower waves
        float top[NT], l[NT], own[NT];
        logits(0);
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            const int r = n0 + nw + 32 * j + (lane & 31);
            const long lab = r < e.R ? label_of(e.labels, r) : -1, at = lab - m0 - mw;
            own[j] = -INFINITY;                                   // the label's logit, where the wave has it
            if (__any(at >= 0 && at < 32 * MT && lab < e.V)) {
                place(lab < e.V ? at : -1, [&](int i, int x) {
                    own[j] = acc[i][j][x];
                    if (mtiles > 1) e.zl[r] = own[j];
                });
            }
            own[j] = attn::half_max(own[j]);
            top[j] = -INFINITY;
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int x = 0; x < 16; ++x) top[j] = fmaxf(top[j], acc[i][j][x]);
            top[j] = attn::half_max(top[j]);
            const float base = top[j] == -INFINITY ? 0.f : top[j];
            l[j] = 0.f;
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int x = 0; x < 16; ++x) l[j] += __builtin_amdgcn_exp2f(acc[i][j][x] - base);
            l[j] = attn::half_sum(l[j]);
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < NT; ++j)
            if (wm && h == 0) { join[nw + 32 * j + lane] = top[j]; join[BN + nw + 32 * j + lane] = l[j]; join[2 * BN + nw + 32 * j + lane] = own[j]; }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            const int r = n0 + nw + 32 * j + lane;
            if (wm || h || r >= e.Rp) continue;
            const float t2 = join[nw + 32 * j + lane], l2 = join[BN + nw + 32 * j + lane], M = fmaxf(top[j], t2), base = M == -INFINITY ? 0.f : M;
            const float L = l[j] * __builtin_amdgcn_exp2f(top[j] - base) + l2 * __builtin_amdgcn_exp2f(t2 - base);
            if (mtiles > 1) {
                e.pm[(long)mt * e.Rp + r] = M;
                e.pl[(long)mt * e.Rp + r] = L;
            } else if (r < e.R) finish_row(e.loss, e.lse_out, r, M, L, fmaxf(own[j], join[2 * BN + nw + 32 * j + lane]), label_of(e.labels, r), e.V);
        }
    } else if constexpr (EPI == E_DZ) {                           // m: vocabulary entries from v0 on, n: rows of x
        const int up = SCALED ? 0 : dz_exp(e);
        logits(e.v0);
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            const int r = n0 + nw + 32 * j + (lane & 31);
            const long lab = r < e.R ? label_of(e.labels, r) : -1;
            const bool has = lab >= 0 && lab < e.V;
            // a row that is left out: p = exp2(-inf) = 0 and g = 0
            const float g = has ? times2(e.dloss[r], SCALED ? dz_exp(e, r) : up) : 0.f, lse = has ? e.lse[r] * LOG2E : INFINITY;
            // (lse is rounded: where it is large an exponent can come out above 0, which no probability's is; a NaN stays one)
            if (__any(has && fabsf(lse) > 1048576.f))
#pragma unroll
                for (int i = 0; i < MT; ++i)
#pragma unroll
                    for (int x = 0; x < 16; ++x) acc[i][j][x] = acc[i][j][x] > lse ? lse : acc[i][j][x];
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int x = 0; x < 16; ++x) acc[i][j][x] = has ? g * __builtin_amdgcn_exp2f(acc[i][j][x] - lse) : 0.f;
            const long at = lab - e.v0 - m0 - mw;
            if (__any(has && at >= 0 && at < 32 * MT)) place(has ? at : -1, [&](int i, int x) { acc[i][j][x] -= g; });
        }
        // through LDS into whole row pieces of the (rows, piece) array; the column sums (db) on the way
        constexpr int E = sizeof(OP), PER = 16 / E, CH = BM / PER, REP = BN * CH / 256;
        static_assert(BN * BM * E <= ST * STAGE && 256 / CH * BM * 4 <= ST * STAGE, "");
        float sum[PER];
#pragma unroll
        for (int k = 0; k < PER; ++k) sum[k] = 0.f;
        int down[REP];
#pragma unroll
        for (int t = 0; t < REP; ++t) down[t] = SCALED && (e.db || e.db_out) ? -dz_exp(e, n0 + (threadIdx.x + 256 * t) / CH) : 0;
#pragma unroll
        for (int p = 0; p < PZ; ++p) {
            __syncthreads();
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int i = 0; i < MT; ++i)
#pragma unroll
                    for (int a = 0; a < 4; ++a) {
                        typename Num<OP>::x4 q;
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            q[x] = (OP)acc[i][j][4 * a + x];
                            if constexpr (PZ == 2) acc[i][j][4 * a + x] -= (float)q[x];
                        }
                        const int c = mw + 32 * i + 8 * a + 4 * h;
                        *reinterpret_cast<typename Num<OP>::x4*>(lds + chunk_at<BM * E>(nw + 32 * j + (lane & 31), c / PER) + c % PER * E) = q;
                    }
            __syncthreads();
#pragma unroll
            for (int t = 0; t < REP; ++t) {
                const int row = (threadIdx.x + 256 * t) / CH, ch = threadIdx.x % CH, r = n0 + row, c = m0 + ch * PER;
                const auto q = *reinterpret_cast<const typename Num<OP>::x16*>(lds + chunk_at<BM * E>(row, ch));
                if (r < e.Rp && c < e.dz_ld) *reinterpret_cast<typename Num<OP>::x16*>(reinterpret_cast<OP*>(e.dz) + p * e.dz_plane + (long)r * e.dz_ld + c) = q;
#pragma unroll
                for (int k = 0; k < PER; ++k) sum[k] += SCALED ? times2((float)q[k], down[t]) : (float)q[k];
            }
        }
        if (e.db || e.db_out) {
            float* red = reinterpret_cast<float*>(lds);           // (256 / CH, BM)
            __syncthreads();
#pragma unroll
            for (int k = 0; k < PER; ++k) red[threadIdx.x / CH * BM + threadIdx.x % CH * PER + k] = sum[k];
            __syncthreads();
            if ((int)threadIdx.x < BM && m0 + (int)threadIdx.x < e.dz_ld) {
                float v = 0.f;
#pragma unroll
                for (int k = 0; k < 256 / CH; ++k) v += red[k * BM + threadIdx.x];
                if constexpr (!SCALED) v = times2(v, -up);
                const int c = m0 + threadIdx.x;
                if (!e.db_out) e.db[(long)nt * e.dz_ld + c] = v;
                else if (e.v0 + c < e.V) e.db_out[c] = (elt)(e.db_accumulate ? (float)e.db_out[c] + v : v);
            }
        }
    } else {
        // (packed: dz's powers are the row's for dx, and in x for dW)
        const int ex = SCALED ? -DZ_BITS - up_exp(max_of(e.parts + (e.with_w ? PART_W : PART_X) * PARTS)) : -dz_exp(e);
        int down[MT][16];
        if constexpr (SCALED) {
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int a = 0; a < 4; ++a) {
                    typedef __attribute__((ext_vector_type(4))) int i32x4;
                    i32x4 g = {0, 0, 0, 0};
                    if (e.with_w) g = *reinterpret_cast<const i32x4*>(e.g_e + m0 + mw + 32 * i + 8 * a + 4 * h);
#pragma unroll
                    for (int c = 0; c < 4; ++c) down[i][4 * a + c] = ex + g[c];
                }
        }
        // every row and column that exists (R, V)
        const auto each = [&](auto&& put) {
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                const int n = n0 + nw + 32 * j + (lane & 31);
                if (n >= e.V) continue;
#pragma unroll
                for (int i = 0; i < MT; ++i)
#pragma unroll
                    for (int x = 0; x < 16; ++x) {
                        const int m = m0 + mw + 32 * i + 8 * (x >> 2) + 4 * h + (x & 3);
                        if (m < e.R) put(m * e.ldo + n, times2(acc[i][j][x], SCALED ? down[i][x] : ex));
                    }
            }
        };
        float* po = reinterpret_cast<float*>(e.out) + sl * e.slice;
        elt* eo = reinterpret_cast<elt*>(e.out);
        if (e.part && e.accumulate) each([&](long at, float v) { po[at] += v; });
        else if (e.part) each([&](long at, float v) { po[at] = v; });
        else if (e.accumulate) each([&](long at, float v) { eo[at] = (elt)((float)eo[at] + v); });
        else each([&](long at, float v) { eo[at] = (elt)v; });
    }
}

// lse and loss of a row from its slices' maxima and sums: 16 rows x 16 groups of slices a block
__global__ __launch_bounds__(256) void finish_kernel(const float* __restrict__ pm, const float* __restrict__ pl, const float* __restrict__ zl, Labels labels,
                                                     float* __restrict__ loss, float* __restrict__ lse, int R, int Rp, int slices) {
    __shared__ float sm[16][17], ss[16][17];
    const int c = threadIdx.x & 15, g = threadIdx.x >> 4, r = blockIdx.x * 16 + c;
    const auto join = [](float& m, float& l, float m2, float l2) {
        const float M = fmaxf(m, m2), base = M == -INFINITY ? 0.f : M;
        l = l * __builtin_amdgcn_exp2f(m - base) + l2 * __builtin_amdgcn_exp2f(m2 - base);
        m = M;
    };
    float m = -INFINITY, l = 0.f;
    if (r < R) {
        int s = g;
        for (; s + 48 < slices; s += 64) {                        // four slices' loads in flight
            float a[4], b[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) { a[k] = pm[(long)(s + 16 * k) * Rp + r]; b[k] = pl[(long)(s + 16 * k) * Rp + r]; }
#pragma unroll
            for (int k = 0; k < 4; ++k) join(m, l, a[k], b[k]);
        }
        for (; s < slices; s += 16) join(m, l, pm[(long)s * Rp + r], pl[(long)s * Rp + r]);
    }
    sm[g][c] = m; ss[g][c] = l;
    __syncthreads();
    if (g || r >= R) return;
#pragma unroll
    for (int x = 1; x < 16; ++x) join(m, l, sm[x][c], ss[x][c]);
    finish_row(loss, lse, r, m, l, zl[r], label_of(labels, r), labels.V);
}

// out (rows, cols) (+)= sum of the slices, for up to three results (blockIdx.y)
struct SumJob { const float* part; elt* out; long slice, ldp, ldo, rows; int slices, cols, accumulate, pad_; };
struct SumJobs { SumJob j[3]; };
__global__ __launch_bounds__(256) void sum_slices_kernel(SumJobs jobs) {
    const SumJob j = jobs.j[blockIdx.y];
    const int across = (j.cols + 255) / 256;
    for (long i = blockIdx.x; i < j.rows * across; i += gridDim.x) {
        const long r = i / across;
        const int c = (int)(i - r * across) * 256 + threadIdx.x;
        if (c >= j.cols) continue;
        float v = 0.f;
        const float* p = j.part + r * j.ldp + c;
        int s = 0;
        for (; s + 8 <= j.slices; s += 8) {                       // eight loads in flight
            float t[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) t[k] = p[(s + k) * j.slice];
#pragma unroll
            for (int k = 0; k < 8; ++k) v += t[k];
        }
        for (; s < j.slices; ++s) v += p[s * j.slice];
        elt* o = j.out + r * j.ldo + c;
        *o = (elt)(j.accumulate ? (float)*o + v : v);
    }
}

// ---- plan of a call: what is packed, the pieces, the tiles, the workspace
struct Plan {
    int Rp, Dp, Vp;                     // rows, hidden width and vocabulary rounded up to the contraction steps
    bool pack_x, pack_w, own_x;         // own_x: dW reads a packing of x of its own
    int piece, pieces;
    bool small_z, small_dx, small_dw;   // 64 x 64 tiles instead of 128 x 128
    // operands of the inputs' type, as they are: more matrix cycles, but neither maxima nor packing.  bf16 where all tiles are small: dz in two bf16
    // planes.  fp32 where the products are small (direct()): the fp32 matrix instructions.
    bool light;
    int dz_planes, g_from;              // (planes of two bytes)
    int dx_slices, dw_slices, lse_slices, db_slices;
    bool dx_parts;
    size_t parts, rows, xo, wo, xg, a, b, zl, dz, dxp, dwp, dbp, bytes;      // offsets
};
static size_t up(size_t n) { return (n + 255) & ~(size_t)255; }
static int up64(int n) { return (n + 63) & ~63; }
static long tiles(int m, int n, int t) { return (long)cdiv(m, t) * cdiv(n, t); }
// 64 x 64 tiles where 128 x 128 ones leave CUs without work
static bool small(int m, int n) { return tiles(m, n, 128) < 256; }
// slices of a contraction whose tiles still do not give every CU two blocks: of eight steps at least
static int cut(long t, int ksteps) {
    const long s = 512 / t, most = ksteps / 8;
    return (int)(s < 1 || most < 1 ? 1 : s < most ? s : most);
}

// fp32: whether the fp32 matrix instructions on the operands as they are cost less than two more launches (maxima, packing) and the bytes those move, 12 for
// each element of x and W.  R x D x V, us direct / packed.  Forward: 20 x 256 x 1000 12 / 16, 2496 x 256 x 1000 21 / 25, 1 x 512 x 20000 27 / 41, 256 x 512 x
// 20000 54 / 54.  Backward, with three products: 20 x 256 x 1000 21 / 24, 500 x 256 x 1000 25 / 29, 2496 x 256 x 1000 58 / 50, 64 x 512 x 20000 64 / 73,
// 128 rows 95 / 89; where W has to be copied all the same (its rows end inside a 16-byte piece), 16 x 512 x 20001: 78 / 70.
static bool direct(const sarVocabCe* a, bool grad) {
    const long work = (a->R + 63L) / 64 * 64 * a->D * a->V, elements = ((long)a->R + a->V) * a->D;
    return SAR_ELT == 0 && work <= (grad ? (1L << 27) + (a->V % 4 ? 0 : 80 * elements) : (1L << 29) + 160 * elements);
}
constexpr int MOST = 1 << 22;
static bool bad(const sarVocabCe* a) {
    return !a || a->R < 1 || a->D < 1 || a->V < 1 || a->R > MOST || a->D > (1 << 16) || a->V > MOST || (a->label_bytes != 4 && a->label_bytes != 8) || a->ldx < a->D || a->ldk < a->V ||
           a->ldx > MOST || a->ldk > MOST || tiles(a->R, a->V, 64) > (1L << 28);
}
static Plan plan(const sarVocabCe* a, bool grad) {
    Plan p = {};
    p.Rp = up64(a->R); p.Dp = up64(a->D); p.Vp = up64(a->V);
    int cols = p.Vp;
    p.light = direct(a, grad);                                    // (64 x 64 tiles in any case)
    if (!grad) {
        p.small_z = p.light || small(a->V, a->R);
        p.lse_slices = cdiv(a->V, p.small_z ? 64 : 128);
    } else {
        // a piece's dz: about 128 MB, which the 256 MB last-level cache holds between its writer and its two readers (8192 x 32000 x 1024: 2384 us;
        // 64 MB 2643, 256 MB 2444, all in one 2408)
        long w = (128L << 20) / ((long)p.Rp * 2 * NPL) / 256 * 256;
        if (w < 256) w = 256;
        p.pieces = cdiv(a->V, w);
        p.piece = (int)(p.pieces == 1 ? p.Vp : cdiv(cdiv(a->V, p.pieces), 256) * 256L);
        p.pieces = cdiv(a->V, p.piece);
        cols = p.piece < p.Vp ? p.piece : p.Vp;
        p.small_z = p.light || small(cols, p.Rp); p.small_dx = p.light || small(a->R, a->D); p.small_dw = p.light || small(a->D, cols);
        p.dx_slices = cut(tiles(a->R, a->D, p.small_dx ? 64 : 128), cols / 32);
        p.dw_slices = cut(tiles(a->D, cols, p.small_dw ? 64 : 128), p.Rp / 32);
        p.db_slices = cdiv(p.Rp, p.small_z ? 64 : 128);
        p.dx_parts = p.dx_slices > 1 || p.pieces > 1;
        p.light |= SAR_ELT == 1 && p.small_z && p.small_dx && p.small_dw;
        p.dz_planes = p.light ? 2 : NPL;
        p.g_from = p.light ? G_ONE : BWD_SCALED ? G_EACH : a->R > G_FEW ? G_PARTS : G_ROWS;
        p.own_x = !p.light && BWD_SCALED && a->dkernel;
    }
    // operands are read where they lie when they have the products' type, their rows start on 4-byte boundaries (what a load into LDS needs) and
    // end with a whole 16-byte piece, or a whole step (Operand: TAIL), where they are read along the contraction (x, and W for dx)
    const bool scaled = !p.light && (grad ? BWD_SCALED : FWD_SCALED);
    constexpr int PIECE = 16 / sizeof(elt), WORD = SAR_ELT == 0 ? 1 : 2;         // elements of 16 bytes, of 4
    p.pack_x = scaled || a->D % (p.small_z ? PIECE : 64) || a->ldx % WORD || (uintptr_t)a->x % 4;
    p.pack_w = scaled || a->V % (!grad ? WORD : p.small_dx ? PIECE : 64) || a->ldk % WORD || (uintptr_t)a->kernel % 4;
    size_t at = 0;
    const auto take = [&](size_t n) { const size_t o = at; at += up(n); return o; };
    p.parts = take(3 * PARTS * 4);
    if (scaled) p.rows = take((size_t)row_places(a->R) * (grad ? 8 : 4));
    if (p.own_x) p.xg = take((size_t)a->R * p.Dp * 2 * NPL);
    if (p.pack_x) p.xo = take((size_t)a->R * p.Dp * 2 * NPL);
    if (p.pack_w) p.wo = take((size_t)a->D * p.Vp * 2 * NPL);
    if (!grad) {
        p.a = take((size_t)p.lse_slices * p.Rp * 4); p.b = take((size_t)p.lse_slices * p.Rp * 4);
        p.zl = take((size_t)p.Rp * 4);
    } else {
        p.dz = take((size_t)p.Rp * cols * 2 * p.dz_planes);
        if (p.dx_parts) p.dxp = take((size_t)p.dx_slices * a->R * a->D * 4);
        if (p.dw_slices > 1) p.dwp = take((size_t)p.dw_slices * a->D * cols * 4);
        if (a->dbias && p.db_slices > 1) p.dbp = take((size_t)p.db_slices * cols * 4);
    }
    p.bytes = at;
    return p;
}

// contraction elements per LDS stage: 64, two stages (whole 128-byte lines where an operand is read along the contraction; half the barriers) -- an 8192 x
// 8192 piece against 1024, us with 64 / with 32: dx 147 / 183, dW 128 / 143, dz 158 / 160.  fp32 (two planes): 32.
// Logits of a shorter contraction on 128 x 128 tiles: 32 with three stages, whose blocks start and end beside two others.  bf16, us with 64 / with 32, D =
// 256, 512, 768, 1024, 2048 (fp16 within 1 % of the same ratios): 777 x 40000 41 / 37, 56 / 53, 71 / 70, 88 / 86, 150 / 157; 4096 x 16000 64 / 56, 93 / 85,
// 119 / 116, 148 / 149, 258 / 284; 8192 x 32000 220 / 188, 320 / 301, 425 / 425, 532 / 553, 986 / 1081.
constexpr int step_of(bool planes = NPL == 2) { return planes ? 32 : 64; }
static int logits_step(const sarVocabCe* a, bool small_tiles) { return small_tiles || a->D > 768 ? step_of() : 32; }
static unsigned some_blocks(long n) { return (unsigned)(n < 1 ? 1 : n < 4096 ? n : 4096); }
// the operands as the products read them; xg: x as dW reads it
struct Operands { Side x, w, xg; };
template <typename OP, bool SCALED> static Operands operands(const sarVocabCe* a, const Plan& p, bool grad, hipStream_t st) {
    char* ws = reinterpret_cast<char*>(a->ws);
    float* parts = reinterpret_cast<float*>(ws + p.parts);
    const float* dloss = grad ? a->dloss : nullptr;
    MaxJobs max = {{}, {a->labels, a->label_bytes, a->V}, dloss};
    int n = 0;
    if (p.own_x) max.j[n++] = {a->x, a->R, a->ldx, a->D, MAX_ROWS, PART_X};
    if (SCALED) max.j[n++] = {a->kernel, a->D, a->ldk, a->V, MAX_ALL, PART_W};
    if (grad && p.g_from == G_PARTS) max.j[n++] = {a->dloss, 1, a->R, a->R, MAX_G, PART_G};
    if (n) hipLaunchKernelGGL(absmax_kernel, dim3(PARTS, n), dim3(1024), 0, st, max, parts);
    Operands o = {{a->x, 0, a->ldx, 0, 0}, {a->kernel, 0, a->ldk, 0, 0}, {}};
    PackJobs jobs = {{}, max.labels, dloss};
    n = 0;
    long blocks = 0;
    const auto pack = [&](Side& s, size_t to, int rows, int cols, int pitch, const float* part, int* row_e, void* all) {
        jobs.j[n++] = {reinterpret_cast<const elt*>(s.p), ws + to, rows, s.ld, (long)rows * pitch, cols, pitch, part, row_e, all};
        s = {ws + to, (long)rows * pitch, pitch, 0, 0};
        const long b = row_e ? cdiv(rows, 4) : (long)rows * cdiv(pitch, 2048);
        blocks = b > blocks ? b : blocks;
    };
    if (p.pack_x) pack(o.x, p.xo, a->R, a->D, p.Dp, p.own_x ? parts + PART_X * PARTS : nullptr, SCALED ? reinterpret_cast<int*>(ws + p.rows) : nullptr, p.own_x ? ws + p.xg : nullptr);
    if (p.pack_w) pack(o.w, p.wo, a->D, a->V, p.Vp, SCALED ? parts + PART_W * PARTS : nullptr, nullptr, nullptr);
    if (n) hipLaunchKernelGGL((pack_kernel<OP, SCALED>), dim3(some_blocks(blocks), n), dim3(256), 0, st, jobs);
    o.xg = o.x;
    if (p.own_x) o.xg.p = ws + p.xg;
    return o;
}
static Job job_of(Side A, Side B, const Epi& e, int m, int n, int k, int step, int slices, bool small_tiles) {
    const int t = small_tiles ? 64 : 128;
    return {A, B, e, cdiv(m, t), cdiv(n, t), cdiv(k, step), slices};
}
static unsigned blocks_of(const Job& j) { return (unsigned)attn::xcd_grid((long)j.mtiles * j.ntiles * j.slices); }
static dim3 grid_of(const Job& j) {
    const unsigned n = blocks_of(j);
    return n <= LAUNCH_ROW ? dim3(n) : dim3(LAUNCH_ROW, (n + LAUNCH_ROW - 1) / LAUNCH_ROW);
}
template <typename OP, bool AD, bool BD, int EPI, bool SCALED> static void product(const Job& j, bool small_tiles, int step, hipStream_t st) {
    constexpr int BK = step_of();
    const dim3 grid = grid_of(j), block(256);
    if (small_tiles) hipLaunchKernelGGL((product_kernel<OP, BK, 1, 1, AD, BD, EPI, SCALED, NPL, NPL, NPL>), grid, block, 0, st, j);
    else if (EPI == E_GRAD || step == BK) hipLaunchKernelGGL((product_kernel<OP, BK, 2, 2, AD, BD, EPI, SCALED, NPL, NPL, NPL>), grid, block, 0, st, j);
    else if constexpr (EPI != E_GRAD) hipLaunchKernelGGL((product_kernel<OP, 32, 2, 2, AD, BD, EPI, SCALED, NPL, NPL, NPL>), grid, block, 0, st, j);
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
    Operands in = p.light ? operands<elt, false>(a, p, false, st) : operands<fwd16, FWD_SCALED>(a, p, false, st);
    Side &x = in.x, &w = in.w;
    w.len = p.pack_w ? p.Vp : a->V; w.k = a->D;
    x.len = a->R; x.k = p.pack_x ? p.Dp : a->D;
    Epi e = {};
    e.parts = reinterpret_cast<float*>(ws + p.parts); e.row_e = reinterpret_cast<int*>(ws + p.rows);
    e.bias = reinterpret_cast<const elt*>(a->bias); e.labels = {a->labels, a->label_bytes, a->V};
    e.pm = reinterpret_cast<float*>(ws + p.a); e.pl = reinterpret_cast<float*>(ws + p.b); e.zl = reinterpret_cast<float*>(ws + p.zl);
    e.R = a->R; e.V = a->V; e.Rp = p.Rp;
    e.loss = a->loss; e.lse_out = a->lse;
    const int step = logits_step(a, p.small_z);
    const Job z = job_of(w, x, e, a->V, a->R, p.Dp, p.light ? 32 : step, 1, p.small_z);
    if constexpr (SAR_ELT == 0) {
        if (p.light) hipLaunchKernelGGL((product_kernel<elt, 32, 1, 1, true, false, E_LSE, false, 1, 1, 1>), dim3(blocks_of(z)), dim3(256), 0, st, z);
    }
    if (!p.light) product<fwd16, true, false, E_LSE, FWD_SCALED>(z, p.small_z, step, st);
    if (z.mtiles > 1) hipLaunchKernelGGL(finish_kernel, dim3((unsigned)cdiv(a->R, 16)), dim3(256), 0, st, e.pm, e.pl, e.zl, e.labels, a->loss, a->lse, a->R, p.Rp, p.lse_slices);
    SAR_CHECK_LAUNCH();
    return SAR_OK;
}

extern "C" int SAR_FN(sar_vocab_ce_bwd)(const sarVocabCe* a, hipStream_t st) {
    if (bad(a) || !a->x || !a->kernel || !a->labels || !a->dloss || !a->lse || !a->ws || (uintptr_t)a->ws % 256 ||
        (!a->dx && !a->dkernel && !a->dbias) || (a->accumulate && SAR_ELT != 0)) return SAR_EINVAL;
    const Plan p = plan(a, true);
    if (a->ws_bytes < 0 || (size_t)a->ws_bytes < p.bytes) return SAR_EINVAL;
    char* ws = reinterpret_cast<char*>(a->ws);
    void* dz = ws + p.dz;
    const Operands in = p.light ? operands<elt, false>(a, p, true, st) : operands<bwd16, BWD_SCALED>(a, p, true, st);
    const auto from = [&](const Side& s, int v) { Side t = s; t.p = reinterpret_cast<const char*>(s.p) + (long)v * (p.light ? (long)sizeof(elt) : 2); return t; };
    for (int i = 0; i < p.pieces; ++i) {
        const int v0 = i * p.piece, cols = a->V - v0 < p.piece ? a->V - v0 : p.piece, ld = up64(cols);
        const long plane = (long)p.Rp * ld;
        Epi e = {};
        e.parts = reinterpret_cast<float*>(ws + p.parts); e.row_e = reinterpret_cast<int*>(ws + p.rows); e.g_e = e.row_e + row_places(a->R);
        e.bias = reinterpret_cast<const elt*>(a->bias); e.labels = {a->labels, a->label_bytes, a->V}; e.dloss = a->dloss; e.lse = a->lse;
        e.dz = dz; e.dz_plane = plane; e.dz_ld = ld;
        if (a->dbias && p.db_slices > 1) e.db = reinterpret_cast<float*>(ws + p.dbp);
        else if (a->dbias) { e.db_out = reinterpret_cast<elt*>(a->dbias) + v0; e.db_accumulate = a->accumulate; }
        e.g_from = p.g_from; e.R_all = a->R;
        e.R = a->R; e.V = a->V; e.v0 = v0; e.Rp = p.Rp;
        Side wz = from(in.w, v0), xz = in.x;
        wz.len = (p.pack_w ? p.Vp : a->V) - v0; wz.k = a->D;
        xz.len = a->R; xz.k = p.pack_x ? p.Dp : a->D;
        const int step = logits_step(a, p.small_z);
        const Job z = job_of(wz, xz, e, ld, p.Rp, p.Dp, step, 1, p.small_z);
        constexpr int PZ = SAR_ELT == 1 ? 2 : 1;                  // planes of the light form's dz
        if constexpr (SAR_ELT != 2) {
            if (p.light) hipLaunchKernelGGL((product_kernel<elt, step_of(), 1, 1, true, false, E_DZ, false, 1, 1, PZ>), dim3(blocks_of(z)), dim3(256), 0, st, z);
        }
        if (!p.light) product<bwd16, true, false, E_DZ, BWD_SCALED>(z, p.small_z, step, st);
        SumJobs sums = {};
        int ns = 0;
        long blocks = 0;
        const auto sum = [&](size_t from_, int slices, long slice, long rows, int cols_, long ldp, elt* out, long ldo, int acc) {
            sums.j[ns++] = {reinterpret_cast<float*>(ws + from_), out, slice, ldp, ldo, rows, slices, cols_, acc, 0};
            const long b = rows * cdiv(cols_, 256);
            blocks = b > blocks ? b : blocks;
        };
        Job dw = {}, dx = {};
        if (a->dkernel) {
            Epi o = e;
            o.R = a->D; o.V = cols; o.with_w = 0; o.part = p.dw_slices > 1;
            const Side A = {in.xg.p, in.xg.plane, in.xg.ld, p.pack_x ? p.Dp : a->D, a->R}, B = {dz, plane, ld, ld, p.Rp};
            elt* out = reinterpret_cast<elt*>(a->dkernel) + v0;
            if (o.part) {
                o.out = ws + p.dwp; o.slice = (long)a->D * ld; o.ldo = ld;
                sum(p.dwp, p.dw_slices, o.slice, a->D, cols, ld, out, a->V, a->accumulate);
            } else { o.out = out; o.ldo = a->V; o.accumulate = a->accumulate; }
            dw = job_of(A, B, o, a->D, cols, p.Rp, step_of(p.dz_planes == 2), p.dw_slices, p.small_dw);
        }
        if (a->dx) {
            Epi o = e;
            o.R = a->R; o.V = a->D; o.with_w = 1; o.ldo = a->D; o.part = p.dx_parts;
            const Side A = {dz, plane, ld, p.Rp, ld}, B = {from(in.w, v0).p, in.w.plane, in.w.ld, a->D, p.pack_w ? ld : cols};
            if (o.part) {
                o.out = ws + p.dxp; o.slice = (long)a->R * a->D; o.accumulate = i > 0;
                if (i == p.pieces - 1) sum(p.dxp, p.dx_slices, o.slice, a->R, a->D, a->D, reinterpret_cast<elt*>(a->dx), a->D, 0);
            } else o.out = a->dx;
            dx = job_of(A, B, o, a->R, a->D, ld, step_of(p.dz_planes == 2), p.dx_slices, p.small_dx);
        }
        const unsigned first = a->dkernel ? blocks_of(dw) : 0, both = first + (a->dx ? blocks_of(dx) : 0);
        if (p.light) {
            if constexpr (SAR_ELT != 2)
                if (both) hipLaunchKernelGGL((grads_kernel<elt, step_of(true), step_of(true), false, 1, PZ>), dim3(both), dim3(256), 0, st, dw, dx, (int)first);
        } else if (a->dkernel && a->dx && p.small_dw && p.small_dx) {
            hipLaunchKernelGGL((grads_kernel<bwd16, step_of(), step_of(), BWD_SCALED, NPL, NPL>), dim3(both), dim3(256), 0, st, dw, dx, (int)first);
        } else {
            if (a->dkernel) product<bwd16, true, true, E_GRAD, BWD_SCALED>(dw, p.small_dw, step_of(), st);
            if (a->dx) product<bwd16, false, false, E_GRAD, BWD_SCALED>(dx, p.small_dx, step_of(), st);
        }
        if (a->dbias && p.db_slices > 1) sum(p.dbp, p.db_slices, ld, 1, cols, ld, reinterpret_cast<elt*>(a->dbias) + v0, cols, a->accumulate);
        if (ns) hipLaunchKernelGGL(sum_slices_kernel, dim3(some_blocks(blocks), ns), dim3(256), 0, st, sums);
    }
    SAR_CHECK_LAUNCH();
    return SAR_OK;
}
