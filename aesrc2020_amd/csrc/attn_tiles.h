// What the attention kernels share: 16-byte fragments, MFMA tiles of 32 x 32, the LDS layout of a (rows, D) tile.
//
// Every product here keeps one side in registers (32 columns n per wave) and streams the other through LDS (32 rows m per step), and is
// written so that its 32 x 32 result can be the next product's operand WITHOUT leaving the registers:
//   * a 32 x 32 result holds column n = lane % 32, rows m = 8 a + 4 h + c (h = lane / 32; a, c = 0..3): sixteen values of ONE column.
//   * as the B operand of the next product (n = lane % 32, contraction index over those rows), the k-th slot of half h may be ANY row as
//     long as the A operand names the same one: with 16-bit types step s takes rows 16 s + {4 h + c, 8 + 4 h + c}, in fp32 step (a, c)
//     takes row 8 a + 4 h + c.  The A operand of that product is the streamed tile read "down its columns": ds_read_b64_tr_b16 hands
//     a lane four consecutive rows of one column (16-bit), plain 4-byte reads do it in fp32.
// A "fragment" is 16 bytes of a row: bytes [32 c + 16 h, +16) of chunk c -- eight 16-bit values (one 32x32x16 MFMA) or four fp32 values
// (four 32x32x2 MFMAs whose k-th pair of dims is {8 c + k, 8 c + 4 + k}).
#pragma once
#include "common.h"

typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(4))) __bf16 bf16x4;
typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(4))) _Float16 f16x4;
typedef __attribute__((ext_vector_type(2))) _Float16 f16x2;
typedef __attribute__((ext_vector_type(4))) short i16x4;
typedef __attribute__((ext_vector_type(4))) unsigned u32x4;
typedef __attribute__((ext_vector_type(2))) unsigned u32x2;

namespace attn {

template <typename T> struct Num;
template <> struct Num<float> { typedef f32x4 x16; typedef f32x4 x4; static constexpr int PER = 4; };
template <> struct Num<__bf16> { typedef bf16x8 x16; typedef bf16x4 x4; static constexpr int PER = 8; };
template <> struct Num<_Float16> { typedef f16x8 x16; typedef f16x4 x4; static constexpr int PER = 8; };

template <typename T> __device__ __forceinline__ typename Num<T>::x16 as16(u32x4 v) { return __builtin_bit_cast(typename Num<T>::x16, v); }

// acc += A B over one 32-byte chunk
template <typename T> __device__ __forceinline__ f32x16 mma(u32x4 a, u32x4 b, f32x16 acc) {
    if constexpr (sizeof(T) == 4) {
        const f32x4 x = as16<float>(a), y = as16<float>(b);
#pragma unroll
        for (int i = 0; i < 4; ++i) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(x[i], y[i], acc, 0, 0, 0);
        return acc;
    } else if constexpr (__is_same(T, __bf16)) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(as16<__bf16>(a), as16<__bf16>(b), acc, 0, 0, 0);
    } else {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(as16<_Float16>(a), as16<_Float16>(b), acc, 0, 0, 0);
    }
}

// bytes between two rows of a tile in LDS: a power of two, so that the swizzle below stays inside the row
template <typename T, int DP> constexpr int pitch() {
    constexpr int b = DP * (int)sizeof(T);
    return b <= 64 ? 64 : b <= 128 ? 128 : b <= 256 ? 256 : 512;
}
// 16-byte chunk `ch` of row `row`: eight consecutive rows put one chunk into eight different bank groups of 16 bytes (row-wise 16-byte
// reads), four consecutive rows put a PAIR of chunks into four different ones (the transposing reads).  LDS hands out sixteen such groups a cycle, so
// this costs twice the fewest cycles.  SIXTEEN (rows of 64 to 256 bytes): sixteen rows, and four rows a run of FOUR chunks, in different groups, no
// conflict left -- for more address arithmetic: the vocabulary products gain 2 % by it; attention's loops, which need the registers, do not (8 x 1024
// x 4096: dQ 391 -> 385 us, dK, dV 565 -> 595; fp32 64 x 72 x 39 28 -> 33).
// (every bit of the swizzle is one bit of the row: the swizzle of a sum of rows without common bits is the two swizzles' xor)
template <int PITCH, bool SIXTEEN = false> __device__ __forceinline__ constexpr int swizzle(int row) {
    if constexpr (SIXTEEN) return PITCH == 64 ? (row >> 2) & 3 : PITCH == 128 ? ((row & 2) << 1) | ((row >> 2) & 3) : ((row & 3) << 2) | ((row >> 2) & 3);
    return PITCH == 64 ? (row & 2) | ((row >> 2) & 1) : ((row & 3) << 1) | ((row >> 2) & 1);
}
template <int PITCH, bool SIXTEEN = false> __device__ __forceinline__ int chunk_at(int row, int ch) { return row * PITCH + ((ch ^ swizzle<PITCH, SIXTEEN>(row)) << 4); }
// fragment of chunk c: row `row`
template <int PITCH> __device__ __forceinline__ u32x4 frag(const char* tile, int row, int c, int h) {
    return *reinterpret_cast<const u32x4*>(tile + chunk_at<PITCH>(row, 2 * c + h));
}
__device__ __forceinline__ u32x2 tr16(const char* p) {
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4*)p));
}

// acc (32 columns-of-the-tile x 32 n) += tile^T P for 32 tile rows starting at row0; dims [32 dt, +32); p: a 32 x 32 result (see above)
// P's planes: 16-bit operands in groups of two fragments (steps s = 0, 1)
template <typename T, int PITCH> __device__ __forceinline__ f32x16 mma_down(const char* tile, int row0, int dt, const u32x4* p, f32x16 acc, int lane) {
    const int h = lane >> 5;
    if constexpr (sizeof(T) == 4) {
        const int d = 32 * dt + (lane & 31);
#pragma unroll
        for (int a = 0; a < 4; ++a) {
            const f32x4 x = as16<float>(p[a]);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int r = row0 + 8 * a + 4 * h + c;
                const float v = *reinterpret_cast<const float*>(tile + chunk_at<PITCH>(r, d >> 2) + ((d & 3) << 2));
                acc = __builtin_amdgcn_mfma_f32_32x32x2f32(v, x[c], acc, 0, 0, 0);
            }
        }
    } else {
        // lane i of a group of 16 reads 8 bytes of row (i / 4), columns 4 (i % 4) ..; it receives column i of those four rows
        const int i = lane & 15, g = (lane >> 4) & 1;
        const int ch = 4 * dt + 2 * g + ((i >> 1) & 1), off = (i & 1) * 8;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const int r = row0 + 16 * s + 4 * h + (i >> 2);
            const u32x2 lo = tr16(tile + chunk_at<PITCH>(r, ch) + off), hi = tr16(tile + chunk_at<PITCH>(r + 8, ch) + off);
            acc = mma<T>(u32x4{lo[0], lo[1], hi[0], hi[1]}, p[s], acc);
        }
    }
    return acc;
}

// a 32 x 32 result as the B operand of mma_down: fp32 as it is (four fragments), 16-bit rounded to nearest even (two).  That rounding, of probabilities
// and of ds, is of the size of the result's own (errors 1.3 to 1.45 times those of one rounding); a second plane for what it drops would double these
// products, half of the forward's and of each gradient's.
template <typename T> __device__ __forceinline__ void pack(const f32x16& s, u32x4* p) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int a = 0; a < 4; ++a) p[a] = __builtin_bit_cast(u32x4, f32x4{s[4 * a], s[4 * a + 1], s[4 * a + 2], s[4 * a + 3]});
    } else {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            typename Num<T>::x16 v;
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = (T)s[8 * k + j];
            p[k] = __builtin_bit_cast(u32x4, v);
        }
    }
}

// the fragments of one row (a wave's column n), zero past D and for rows that do not exist
template <typename T, int DP> __device__ __forceinline__ void load_row(const T* p, bool ok, int D, int h, u32x4* f, bool negate = false) {
    constexpr int NC = DP * (int)sizeof(T) / 32;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        const int d = (2 * c + h) * Num<T>::PER;
        f[c] = u32x4{0, 0, 0, 0};
        if (ok && d < D) f[c] = *reinterpret_cast<const u32x4*>(p + d);
        if (negate) f[c] = f[c] ^ (sizeof(T) == 4 ? 0x80000000u : 0x80008000u);
    }
}

// v of the lower and of the upper half of a column (lanes l and l ^ 32), to both.  (Written out: hipcc 7.2 takes the two results of its builtin for
// one.  The wait states are those it puts between a VALU write of an operand and the swap.)
__device__ __forceinline__ void halves(float v, float& lo, float& hi) {
    lo = v; hi = v;
    asm("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(lo), "+v"(hi));
}
__device__ __forceinline__ float half_max(float v) { float a, b; halves(v, a, b); return fmaxf(a, b); }
__device__ __forceinline__ float half_sum(float v) { float a, b; halves(v, a, b); return a + b; }

// ---- tiles straight from memory into LDS.  A buffer descriptor over the rows that exist makes the hardware deliver zeros for all others (no
// branches, no clamps, and a row behind a length can hold anything); the lanes' 16-byte pieces land in LDS in lane order, so the swizzle is
// applied to WHICH piece a lane fetches.
__device__ __forceinline__ unsigned lds_addr(const void* p) { return (unsigned)(uintptr_t)(__attribute__((address_space(3))) const char*)p; }
__device__ __forceinline__ u32x4 descriptor(const void* base, unsigned bytes) {
    const uintptr_t b = (uintptr_t)base;
    return u32x4{(unsigned)__builtin_amdgcn_readfirstlane((int)(unsigned)b), (unsigned)__builtin_amdgcn_readfirstlane((int)(unsigned)(b >> 32)) & 0xffffu,
                 (unsigned)__builtin_amdgcn_readfirstlane((int)bytes), 0x00027000u};
}
// (m0 is put back: the compiler does not know that the statement uses it.  The loads are waited for with tile_barrier().)
__device__ __forceinline__ void dma16(u32x4 rsrc, unsigned offset, unsigned lds) {
    unsigned keep;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tbuffer_load_dwordx4 %2, %3, 0 offen lds\n\ts_mov_b32 m0, %0"
                 : "=&s"(keep) : "s"(lds), "v"(offset), "s"(rsrc) : "memory");
}
// this wave's tile loads have arrived, its LDS reads are done, and so are every other wave's of the block
__device__ __forceinline__ void tile_barrier() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// ROWS rows of `bytes` useful bytes each, `stride` bytes apart, by the block's four waves
template <int PITCH, int ROWS, bool SIXTEEN = false> struct TileLoader {
    static_assert(!SIXTEEN || PITCH <= 256, "a step of the loader is sixteen rows at least");
    static constexpr int CPR = PITCH / 16, ALL = ROWS * PITCH / 1024, N = (ALL + 3) / 4;
    unsigned first, step;
    __device__ __forceinline__ TileLoader(unsigned stride, unsigned bytes) {
        const int slot = threadIdx.x, row = slot / CPR, pos = slot % CPR;
        const unsigned ch = pos ^ swizzle<PITCH, SIXTEEN>(row);   // the piece that belongs at `pos`
        first = ch * 16 < bytes ? row * stride + ch * 16 : 0x80000000u;                        // behind the row: out of any range
        step = 256 / CPR * stride;
    }
    // `rows` of the tile's rows exist (none: zeros)
    __device__ __forceinline__ void load(const void* base, int rows, unsigned stride, unsigned bytes, char* tile, int wave) const {
        const u32x4 rsrc = descriptor(base, rows > 0 ? (unsigned)(min(rows, ROWS) - 1) * stride + bytes : 0);
        const unsigned dst = lds_addr(tile);
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (ALL % 4 == 0 || 4 * i + wave < ALL) dma16(rsrc, first + i * step, dst + (4 * i + wave) * 1024);
    }
};

// the same for one wave alone: 32 rows, waited for with the wave's own count of loads
template <int PITCH> struct WaveLoader {
    static constexpr int CPR = PITCH / 16, RPI = 64 / CPR, N = 32 / RPI;
    unsigned row, piece;
    __device__ __forceinline__ WaveLoader(unsigned stride) {
        const int lane = threadIdx.x & 63, r = lane / CPR;
        row = r * stride;
        piece = lane % CPR ^ swizzle<PITCH>(r);
    }
    __device__ __forceinline__ void load(const void* base, int rows, unsigned stride, unsigned bytes, unsigned dst) const {
        const u32x4 rsrc = descriptor(base, rows > 0 ? (unsigned)(min(rows, 32) - 1) * stride + bytes : 0);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const unsigned at = (piece ^ swizzle<PITCH>(i * RPI)) * 16;
            dma16(rsrc, at < bytes ? row + i * RPI * stride + at : 0x80000000u, dst + i * 1024);
        }
    }
};

// blockIdx -> work item such that consecutive items (which share keys and values) land on ONE of the eight XCDs, whose L2 then holds them;
// the grid is rounded up to a multiple of 8, surplus blocks get -1
__device__ __forceinline__ int xcd_item(int n, int block) {
    const int per = (n + 7) >> 3, at = block >> 3, i = (block & 7) * per + at;
    return at < per && i < n ? i : -1;
}
__device__ __forceinline__ int xcd_item(int n) { return xcd_item(n, blockIdx.x); }
static inline long xcd_grid(long n) { return ((n + 7) >> 3) << 3; }

}  // namespace attn
