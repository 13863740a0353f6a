// Tile machinery shared by the attention kernels (gfx950): LDS images of 64 x 64 bf16 tiles filled by LDS-DMA, fragment
// reads of them in both directions, accumulator tiles as operands of the next product, row-wise output staging.
#pragma once
#include "common.h"

#define AT_D 64
#define AT_T 64           // tile length along the streamed sequence
#define AT_BR 128         // rows of the owned sequence per workgroup
#define AT_RING 3         // tiles in LDS per streamed operand
#define AT_TILE (AT_T * AT_D)
#define AT_NEG (-1.0e30f)

typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((address_space(3))) void at_lds_void;
typedef const __attribute__((address_space(1))) void at_global_cvoid;

// 2^x by the bare hardware instruction: arguments here are bounded above and results below 2^-126 may flush to zero
__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// Exchange between lane l and lane l ^ 32 (the two lanes that share a row of a 32x32 accumulator tile): after
// v_permlane32_swap of two copies of v, one copy holds the lower half's values in both halves and the other the
// upper half's, so one max / add finishes the reduction on the vector ALU.
__device__ __forceinline__ void swap_rows32(float& a, float& b) { asm volatile("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(a), "+v"(b)); }
__device__ __forceinline__ float other_half_max(float v) {
    float a = v, b = v;
    swap_rows32(a, b);
    return fmaxf(a, b);
}
__device__ __forceinline__ float other_half_sum(float v) {
    float a = v, b = v;
    swap_rows32(a, b);
    return a + b;
}

// ------------------------------------------------------------------------------------------------
// LDS image of a 64 x 64 bf16 tile: [row][128 B], the 16-byte slots of row r XOR-ed with
//   swz(r) = 4 * ((r >> 1) & 1) + ((r >> 2) & 3).
// Row reads (ds_read_b128, 32 rows per instruction, serviced in the lane groups {0-3, 12-15, 20-27} and
// {4-11, 16-19, 28-31} of each half wave): the 8 rows of equal parity in a group get 8 different slots.
// Transposed reads (ds_read_b64_tr_b16, a half wave reads a 4-row x 32-column block): rows r and r + 2 differ in
// bit 2 of the slot, rows r and r + 1 in the 128-byte parity, so the block covers all 64 banks once.
// The image of an LDS-DMA piece is lane-linear (lane -> row lane / 8, slot lane % 8), so the permutation is applied
// to the source address: slot s of row r receives chunk s ^ swz(r).  Rows past the end of the sequence repeat the
// last row: their scores are masked, and the data stays finite.
// ------------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t at_swz(uint32_t row) { return (((row >> 1) & 1) << 2) | ((row >> 2) & 3); }

struct TileDma {
    uint32_t row[2];  // row of the tile this lane fetches in each of its wave's two pieces (8 pieces of 8 rows per tile)
    uint32_t off[2];  // element offset of the lane's source chunk inside the row
};

__device__ __forceinline__ TileDma tile_dma_setup(int wave, int lane) {
    TileDma d;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const uint32_t row = (2 * wave + j) * 8 + (lane >> 3), slot = lane & 7;
        d.row[j] = row;
        d.off[j] = (slot ^ at_swz(row)) << 3;
    }
    return d;
}

// rows [r0, r0 + 64) of a [*, row_stride] matrix (clamped to last_row) into one tile; two LDS-DMA instructions per wave
__device__ __forceinline__ void tile_dma_issue(const TileDma& d, const bf16* base, uint32_t row_stride, int r0, int last_row, bf16* tile,
                                               int wave) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const uint32_t off = static_cast<uint32_t>(min(r0 + static_cast<int>(d.row[j]), last_row)) * row_stride;
        __builtin_amdgcn_global_load_lds((at_global_cvoid*)(base + off + d.off[j]), (at_lds_void*)(tile + (2 * wave + j) * 512), 16, 0, 0);
    }
}

// Per-lane addressing of the fragment reads (LDS byte offsets inside a tile).
struct FragAddr {
    uint32_t row[4];    // row-major A fragment of k-step ks, row lane % 32 (+ 4096 per 32-row tile)
    uint32_t tr[2][2];  // transposed A fragment: [column tile dt][4-row block blk] (+ 2048 per 16 rows)
};

__device__ __forceinline__ FragAddr frag_addr_setup(int lane) {
    FragAddr f;
    const int hi = lane >> 5, lq = lane & 31, l16 = lane & 15, half = (lane >> 4) & 1, piece = l16 & 3;
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) f.row[ks] = lq * 128 + (((2 * ks + hi) ^ at_swz(lq)) << 4);
#pragma unroll
    for (int dt = 0; dt < 2; ++dt)
#pragma unroll
        for (int blk = 0; blk < 2; ++blk) {
            const uint32_t row = 4 * hi + (l16 >> 2) + 8 * blk;
            const uint32_t slot = (4 * dt + 2 * half + (piece >> 1)) ^ at_swz(row);
            f.tr[dt][blk] = row * 128 + (slot << 4) + (piece & 1) * 8;
        }
    return f;
}

// Every LDS read of a kernel that has LDS-DMA in flight is inline assembly: the compiler cannot tell an ordinary LDS
// load from the pending DMA writes and would drain the whole DMA queue (vmcnt(0)) in front of it, which takes away
// the two tiles of prefetch.  Completion is therefore awaited by hand: LDS reads return in order, so a counted
// lgkmcnt(N) releases all but the youngest N; the scheduling fence keeps the consumers behind the wait.
typedef __attribute__((ext_vector_type(4))) uint32_t u32x4;

template <int N>
__device__ __forceinline__ void lds_wait() {
    asm volatile("s_waitcnt lgkmcnt(%0)" ::"n"(N) : "memory");
    __builtin_amdgcn_sched_barrier(0);
}

// A[i][k] = tile[32 rt + i][16 ks + k], ks = 0..3: rows of the tile as four 32 x 16 A operands (4 reads)
struct RowFrags {
    u32x4 v[4];
};
__device__ __forceinline__ void frag_rows_issue(RowFrags& f, uint32_t tile_lds, const FragAddr& fa, int rt) {
#pragma unroll
    for (int ks = 0; ks < 4; ++ks)
        asm volatile("ds_read_b128 %0, %1 offset:%2" : "=v"(f.v[ks]) : "v"(tile_lds + fa.row[ks]), "n"(4096 * rt) : "memory");
}
__device__ __forceinline__ bf16x8 frag_rows_get(const RowFrags& f, int ks) { return __builtin_bit_cast(bf16x8, f.v[ks]); }

// four consecutive floats of a per-row vector in LDS (the same address in every lane of a half wave: a broadcast)
__device__ __forceinline__ void lds_read_f32x4(f32x4& v, uint32_t addr) { asm volatile("ds_read_b128 %0, %1" : "=v"(v) : "v"(addr) : "memory"); }

// Transposed A fragments of column tile dt for the two 16-row steps j of row tile rt (4 reads):
// A[i][k] = tile[32 rt + 16 j + row(k)][32 dt + i], where row(k) follows the accumulator row order of the 32x32
// MFMA, so that registers 8 j .. 8 j + 7 of a packed accumulator tile are the matching B operand.
struct TrFrags {
    s16x4 lo[2], hi[2];
};
__device__ __forceinline__ void frag_tr_issue(TrFrags& v, uint32_t tile_lds, const FragAddr& fa, int dt, int rt) {
    const uint32_t a0 = tile_lds + fa.tr[dt][0], a1 = tile_lds + fa.tr[dt][1];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        asm volatile("ds_read_b64_tr_b16 %0, %1 offset:%2" : "=v"(v.lo[j]) : "v"(a0), "n"((32 * rt + 16 * j) * 128) : "memory");
        asm volatile("ds_read_b64_tr_b16 %0, %1 offset:%2" : "=v"(v.hi[j]) : "v"(a1), "n"((32 * rt + 16 * j) * 128) : "memory");
    }
}
__device__ __forceinline__ bf16x8 frag_tr_get(const TrFrags& v, int j) {
    const s16x8 r = {v.lo[j][0], v.lo[j][1], v.lo[j][2], v.lo[j][3], v.hi[j][0], v.hi[j][1], v.hi[j][2], v.hi[j][3]};
    return __builtin_bit_cast(bf16x8, r);
}

// registers 8 j .. 8 j + 7 of an accumulator tile as the B operand of the next product
__device__ __forceinline__ bf16x8 pack_half(const f32x16& a, int j) {
    bf16x8 r;
#pragma unroll
    for (int e = 0; e < 8; ++e) r[e] = f32_to_bf16(a[8 * j + e]);
    return r;
}

__device__ __forceinline__ uint32_t lds_addr(const void* p) { return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((at_lds_void*)p)); }

// acc^T[column][row] (two 32-column tiles, the row on the lane) times `mult` -> bf16 rows of 64 in a wave-private LDS
// area (16-byte slots XOR-ed by row & 7), then whole 128-byte rows to global memory: dst(row) is the row's address.
template <typename DstFn>
__device__ __forceinline__ void store_rows32(bf16* so, const f32x16* acc, float mult, int lane, int rows_valid, DstFn dst) {
    const int hi = lane >> 5, lq = lane & 31;
#pragma unroll
    for (int dt = 0; dt < 2; ++dt)
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
            bf16x4 v;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = f32_to_bf16(acc[dt][4 * r4 + e] * mult);
            *reinterpret_cast<bf16x4*>(so + lq * AT_D + (((4 * dt + r4) ^ (lq & 7)) << 3) + 4 * hi) = v;
        }
#pragma unroll
    for (int pass = 0; pass < 4; ++pass) {
        const int row = pass * 8 + (lane >> 3), slot = lane & 7;
        const bf16x8 v = *reinterpret_cast<const bf16x8*>(so + row * AT_D + ((slot ^ (row & 7)) << 3));
        if (row < rows_valid) *reinterpret_cast<bf16x8*>(dst(row) + slot * 8) = v;
    }
}
