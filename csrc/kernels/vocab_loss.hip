// Losses over a large vocabulary (gfx950): cross-entropy behind the output projection, and the divergence of a student's
// distribution from a teacher's top logits, on given logits or behind the projection.
//
// Every loss here is, per row with logits z and q = softmax(z / tau), a weighted cross-entropy against a few targets,
//     L = tau^2 ( sum_k p_k ln p_k - sum_k p_k z[id_k] / tau + lse(z / tau) ),      dL/dz = tau (q - p),      sum_k p_k = 1,
// averaged over the rows that have a target: labels are one target of weight 1 (tau = 1), a teacher gives
// p = softmax(top logits / tau).  Exponents are kept in units of log2.
//
// Behind a projection z = W x the logits never exist as such.  The vocabulary is worked off in tiles: the scores kernel
// holds a 256 x 256 tile of z in fp32 registers and leaves, per row and group of 64 vocabulary entries, the maximum and
// the sum of 2^(z - maximum) in fp32 and (training) the exponentials themselves in bf16 - relative to their group's
// maximum, so the rounding (2^-8 at most) is relative to the value however small the probability.  Once a row's groups
// are joined, one pass turns the exponentials into q - p in place (at the targets from their scores in fp32, see
// vl_target_scores), and two more products give dx = (q - p) W and
// dW = (q - p)^T x; the factor tau / rows is applied to their fp32 sums.
#include "common.h"
#include <type_traits>

typedef __attribute__((address_space(3))) void vl_lds_void;
typedef const __attribute__((address_space(1))) void vl_global_cvoid;

#define VL_INF __builtin_inff()
#define VL_GROUP 64   // vocabulary entries that share a maximum
#define VL_MAX_TOP 1024
#define VL_MAX_ROWS ((1 << 22) - 63)  // rows stay below: rounded up to 64, with up to 1024 threads each, a launch has fewer than 2^32

// A buffer far larger than the caches is written around them: 8192 x 50257 bf16, loss and gradients 2346 -> 2266 us, distillation
// on logits 393 -> 377 us, 2048 rows 544 -> 537 us.  One that the caches hold is read again from them: 512 rows 188 us, written
// around them 191; 64 rows 103 and 105.
#define VL_STREAM_BYTES (64ll << 20)
template <typename V>
__device__ __forceinline__ void vl_store(V* at, V v, bool stream) {
    if (stream) {
        // (the empty statements keep the two stores from being merged into one, which loses the cache policy)
        asm volatile("" ::: "memory");
        __builtin_nontemporal_store(v, at);
        asm volatile("" ::: "memory");
    } else {
        *at = v;
    }
}

__device__ __forceinline__ float vl_exp2(float x) { return __builtin_amdgcn_exp2f(x); }
#define VL_LOG2E 1.4426950408889634f
#define VL_LN2 0.6931471805599453f

// ------------------------------------------------------------------------------------------------
// matrix products:  C[m][n] = sum_k A(m, k) B(n, k), 256 x 256 tiles, 8 waves (2 x 4), K-steps of 64
// An operand is stored with k along its rows ("K-contiguous", [m][k]) or across them ("K-major", [k][m]).
//   KIND 0 scores: A = x [rows][k], B = W [vocab][k]          KIND 1 dx: A = D [rows][vocab], B = W (K-major)
//   KIND 2 dW:     A = D (K-major), B = x (K-major)
// LDS images: K-contiguous [256][64], the 16-byte slots of a row XOR-ed with row & 7; K-major [64][256], the 32-byte units
// of a row XOR-ed with (row & 3) | (row & 8) / 2, so that the rows {8g .. 8g + 3} two lane groups of a transposed read
// touch at once fall on different banks.  The transposed reads take rows 8g .. 8g + 7 for lane group g, the k order of an
// ordinary fragment, so the two kinds of operand go together.
//
// Schedule: a K-step is four phases of 16 MFMAs, each between two barriers, and the two wave rows run one barrier apart:
// on every SIMD one wave's MFMAs cover the other's fragment reads and LDS-DMA requests.  Operands arrive in units of a
// quarter stage, one per phase, six units ahead; a counted wait leaves four in flight.  Workgroups are persistent, so the
// next tile's operands are on their way while a tile is written.
//   A K-contiguous: a phase takes one half of the wave's rows (i) and one part of B - half the columns (B K-contiguous) or
//     one 32-deep slice (B K-major); units {A lower, B part 0, B part 1, A upper}, phases (lower, 0) (lower, 1) (upper, 1) (upper, 0).
//   A K-major: phases (slice, half of the rows); units {B slice 0, A slice 0, B slice 1, A slice 1}.
// A unit is overwritten at least a phase behind its last reader's MFMAs in either order, for either wave row.
//
// Work: whole tiles first, a multiple of the workgroups; the tiles left over (all, where the tiles are few) are cut along k
// into parts that fill the last round, summed in order by vocab_join_kernel.
//
// Measured (a library product of 8192^3 in bf16 runs at 1.5 PFLOP/s): 8192 rows, 50257 entries, width 1024: scores 750 to 800 us by
// the card (1.1 PFLOP/s: 16 K-steps, then exponentials, maxima and 128 KB of results per tile), dx and dW 635 to 680 us (1.3);
// 130001 entries, width 2048: 3.5, 3.1 and 3.2 ms (1.25, 1.4, 1.36).  Bound by the matrix pipe between the tiles' ends.  512 rows,
// width 768: 54, 43 and 51 us; 64 rows, scores alone: 22 us, W read at 3.5 TB/s.
// ------------------------------------------------------------------------------------------------
struct VocabGemm {
    const bf16 *a, *b;
    long long lda, ldb;
    int M, N, K;             // K-contiguous operands hold K rounded up to 64 per row, a K-major A that many rows
    int tiles_m, tiles_n;
    int whole, left, parts;  // units: `whole` tiles, then `left` tiles in `parts` parts each
    int part_steps;
    // scores
    float2* stats;           // [M][groups] {maximum (log2 units), sum}
    bf16* e;                 // [M][lde] exponentials, or nullptr
    long long lde;
    int groups;
    bool stream;
    float scale_log2;        // log2(e) / tau
    // dx, dW
    const float* alpha;      // device factor of the result
    bf16* out;               // bf16 result, or nullptr
    float* out32;            // fp32 result
    long long ldo;
    int accumulate;          // add to out32
    float* part;             // [left][parts][32][512][4]: accumulators as the threads hold them
};

struct RowFrag {
    u32x4 v;
};
struct TrFrag {
    s16x4 lo, hi;
};
template <int OFF>
__device__ __forceinline__ void vl_read(RowFrag& f, uint32_t at) { asm volatile("ds_read_b128 %0, %1 offset:%2" : "=v"(f.v) : "v"(at), "n"(OFF) : "memory"); }
template <int OFF>
__device__ __forceinline__ void vl_read(TrFrag& f, uint32_t at) {
    asm volatile("ds_read_b64_tr_b16 %0, %1 offset:%2" : "=v"(f.lo) : "v"(at), "n"(OFF) : "memory");
    asm volatile("ds_read_b64_tr_b16 %0, %1 offset:%2" : "=v"(f.hi) : "v"(at), "n"(OFF + 4 * 256 * 2) : "memory");
}
// f(0), f(1), ... with compile-time indexes
template <int N, typename F>
__device__ __forceinline__ void vl_for(F f) {
    if constexpr (N > 0) {
        vl_for<N - 1>(f);
        f(std::integral_constant<int, N - 1>{});
    }
}
// the values of reads issued above, taken over behind the wait for them: nothing that uses them can move in front of it
__device__ __forceinline__ bf16x8 vl_take(RowFrag& f) {
    asm volatile("" : "+v"(f.v));
    return __builtin_bit_cast(bf16x8, f.v);
}
__device__ __forceinline__ bf16x8 vl_take(TrFrag& f) {
    asm volatile("" : "+v"(f.lo), "+v"(f.hi));
    const s16x8 v = {f.lo[0], f.lo[1], f.lo[2], f.lo[3], f.hi[0], f.hi[1], f.hi[2], f.hi[3]};
    return __builtin_bit_cast(bf16x8, v);
}
template <int N>
__device__ __forceinline__ void vl_wait_lds() {
    asm volatile("s_waitcnt lgkmcnt(%0)" ::"n"(N) : "memory");
    __builtin_amdgcn_sched_barrier(0);
}

// v of this lane and of lane ^ 16 (or ^ 32), in either order, on the vector ALU
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
template <int LANES>
__device__ __forceinline__ void vl_both(float v, float& a, float& b) {
    const uint32_t x = __builtin_bit_cast(uint32_t, v);
    u32x2 r;
    if constexpr (LANES == 16) r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    else r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    const uint32_t lo = r[0], hi = r[1];  // (a bit cast of a vector's element itself reads element 0)
    a = __builtin_bit_cast(float, lo);
    b = __builtin_bit_cast(float, hi);
}
__device__ __forceinline__ float vl_max4(float v) {  // over lanes l, l ^ 16, l ^ 32, l ^ 48
    float a, b;
    vl_both<16>(v, a, b);
    vl_both<32>(fmaxf(a, b), a, b);
    return fmaxf(a, b);
}
__device__ __forceinline__ float vl_sum4(float v) {
    float a, b;
    vl_both<16>(v, a, b);
    vl_both<32>(a + b, a, b);
    return a + b;
}

template <bool KMAJOR>
__device__ __forceinline__ int vl_swz(int row) { return KMAJOR ? (row & 3) | ((row >> 1) & 4) : row & 7; }

// (tile row, tile column) in groups of eight rows of tiles: the 32 tiles an XCD works on at a time share 8 A and 4 B panels
__device__ __forceinline__ void vl_tile(const VocabGemm& p, int u, int& m0, int& n0) {
    const int per = 8 * p.tiles_n, grp = u / per, gm = min(8, p.tiles_m - grp * 8), in = u - grp * per;
    m0 = (grp * 8 + in % gm) * 256;
    n0 = (in / gm) * 256;
}

template <int KIND>
__global__ __launch_bounds__(512) void vocab_gemm_kernel(const VocabGemm p) {
    constexpr bool A_KM = KIND == 2, B_KM = KIND != 0;
    constexpr int STAGE = 2 * 256 * 64;  // elements: [A tile | B tile]
    extern __shared__ __attribute__((aligned(1024))) bf16 vl_smem[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave >> 2, wn = wave & 3;
    const int r16 = lane & 15, g4 = lane >> 4;
    bf16* stage = vl_smem + 2 * STAGE + wave * (16 * 64);  // 16 rows of the wave's result at a time, as whole 128-byte rows
    const int steps_all = (p.K + 63) / 64, units = p.whole + p.left * p.parts, G = gridDim.x;
    const int first = xcd_remap(blockIdx.x, G);
    float alpha = 1.f;
    if constexpr (KIND != 0) alpha = p.alpha[0];

    struct Unit {
        int m0, n0, k0, steps, part;  // part: -1 for a whole tile, else its place in p.part
    };
    auto unit_of = [&](int u) {
        Unit r;
        if (u < p.whole) {
            vl_tile(p, u, r.m0, r.n0);
            r.k0 = 0;
            r.steps = steps_all;
            r.part = -1;
        } else {
            const int v = u - p.whole, s = v / p.left, t = v - s * p.left;  // parts of one k range side by side: they share operand rows
            vl_tile(p, p.whole + t, r.m0, r.n0);
            r.k0 = s * p.part_steps * 64;
            r.steps = min(p.part_steps, steps_all - s * p.part_steps);
            r.part = t * p.parts + s;
        }
        return r;
    };

    // ---- loader: wave-uniform base per operand, advanced by a K-step, and this lane's byte offset per DMA piece.  Pieces 2i'
    // and 2i' + 1 of a wave belong to staging unit i' of their operand.
    const char *a_base, *b_base;
    uint32_t a_off[4], b_off[4];
    int ld_u = first, ld_s = 0, ld_steps = 0, ld_slot = 0, ld_k = 0;
    auto a_row = [&](int i) {
        const int q = 2 * wave + (i & 1);
        return A_KM ? (i >> 1) * 32 + q * 2 : (q >> 3) * 128 + (i >> 1) * 64 + (q & 7) * 8;
    };
    auto b_row = [&](int i) {
        const int q = 2 * wave + (i & 1);
        return B_KM ? (i >> 1) * 32 + q * 2 : (q >> 2) * 64 + (i >> 1) * 32 + (q & 3) * 8;
    };
    auto lane_off = [&](int row0, long long ld, int origin, int count, bool km) -> uint32_t {
        if (km) {
            const int row = row0 + (lane >> 5), pc = lane & 31;
            const int col = (((pc >> 1) ^ vl_swz<true>(row)) << 4) | ((pc & 1) << 3);
            const int c = min(origin + col, (count - 1) & ~7) - origin;  // (rows hold whole chunks of eight)
            return (static_cast<uint32_t>(row) * static_cast<uint32_t>(ld) + c) * 2u;
        }
        const int row = row0 + (lane >> 3), slot = lane & 7;
        return (static_cast<uint32_t>(min(origin + row, count - 1) - origin) * static_cast<uint32_t>(ld) + ((slot ^ vl_swz<false>(row)) << 3)) * 2u;
    };
    auto load_unit = [&](int u) {
        const Unit r = unit_of(u < units ? u : first);  // (past its last unit the loader repeats the first: nothing reads it)
        a_base = reinterpret_cast<const char*>(p.a + (A_KM ? r.k0 * p.lda + r.m0 : r.m0 * p.lda + r.k0));
        b_base = reinterpret_cast<const char*>(p.b + (B_KM ? r.k0 * p.ldb + r.n0 : r.n0 * p.ldb + r.k0));
        ld_steps = r.steps;
        ld_k = r.k0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            a_off[i] = lane_off(a_row(i), p.lda, r.m0, p.M, A_KM);
            b_off[i] = lane_off(b_row(i), p.ldb, r.n0, p.N, B_KM);
        }
    };
    auto load_a = [&](int half) {
        bf16* tile = vl_smem + ld_slot * STAGE;
#pragma unroll
        for (int i = 2 * half; i < 2 * half + 2; ++i)
            __builtin_amdgcn_global_load_lds((vl_global_cvoid*)(a_base + a_off[i]), (vl_lds_void*)(tile + a_row(i) * (A_KM ? 256 : 64)), 16, 0, 0);
    };
    auto load_b = [&](int half) {
        bf16* tile = vl_smem + ld_slot * STAGE + 256 * 64;
#pragma unroll
        for (int i = 2 * half; i < 2 * half + 2; ++i) {
            uint32_t off = b_off[i];
            if constexpr (KIND == 1) {
                // rows of W beyond the vocabulary repeat its last one (their products are with zeros)
                const int over = ld_k + b_row(i) + (lane >> 5) - (p.K - 1);
                off -= static_cast<uint32_t>(max(over, 0)) * static_cast<uint32_t>(p.ldb) * 2u;
            }
            __builtin_amdgcn_global_load_lds((vl_global_cvoid*)(b_base + off), (vl_lds_void*)(tile + b_row(i) * (B_KM ? 256 : 64)), 16, 0, 0);
        }
    };
    auto load = [&](int r) {  // staging unit r of the K-step under the cursor
        if constexpr (A_KM) {
            if (r & 1) load_a(r >> 1);
            else load_b(r >> 1);
        } else {
            if (r == 0 || r == 3) load_a(r == 3);
            else load_b(r - 1);
        }
        if (r == 3) {
            ld_slot ^= 1;
            a_base += A_KM ? 64 * 2 * p.lda : 64 * 2;
            b_base += B_KM ? 64 * 2 * p.ldb : 64 * 2;
            ld_k += 64;
            if (++ld_s == ld_steps) {
                ld_s = 0;
                ld_u += G;
                load_unit(ld_u);
            }
        }
    };

    // ---- fragment addresses (LDS bytes): a lane constant per operand, the rest as immediate offsets; the stage is bit 16
    // (the kernel has no other LDS, so its dynamic part starts at 0).
    // K-contiguous: rows 16 i + (lane & 15) of the wave's part at i * 2048, the second 32-deep slice with bit 6 turned.
    // K-major: columns 16 i .. + 15 with i << 5 XOR-ed in, slices 16384 apart.
    const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((vl_lds_void*)vl_smem));
    const int tr_row = 8 * g4 + ((lane >> 2) & 3);  // (rows row and row + 4 are swizzled alike)
    const uint32_t row_lane = r16 * 128 + ((g4 ^ (r16 & 7)) << 4), tr_lane = tr_row * 512 + (vl_swz<true>(tr_row) << 5) + 8 * (lane & 3);
    uint32_t at_a = lds0 + (A_KM ? tr_lane ^ (wm << 8) : row_lane + wm * 16384), at_b = lds0 + (B_KM ? tr_lane ^ (wn << 7) : row_lane + wn * 8192);
    constexpr int B_AT = 256 * 64 * 2;

    f32x4 acc[8][4];
    const f32x4 zero4 = {0.f, 0.f, 0.f, 0.f};
    auto enter = [&]() {  // the unit the next phase reads has landed; everybody's waits meet
        asm volatile("s_waitcnt vmcnt(8)\n\ts_barrier" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_setprio(1);
    };
    auto leave = [&]() {
        __builtin_amdgcn_s_setprio(0);
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("s_barrier" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
    };
    using C0 = std::integral_constant<int, 0>;
    using C1 = std::integral_constant<int, 1>;
    auto step = [&](auto first_step) {
        constexpr bool FIRST = decltype(first_step)::value;
        if constexpr (KIND == 0) {
            RowFrag fa[2][4], fb[2][2][2];  // [kk][i], [part][kk][j]
            bf16x8 b[2][2][2];
            auto take_b = [&](int part, int kk) {
                b[part][kk][0] = vl_take(fb[part][kk][0]);
                b[part][kk][1] = vl_take(fb[part][kk][1]);
            };
            auto read_a = [&](auto half) {
                vl_for<8>([&](auto n) { vl_read<(half * 4 + n % 4) * 2048>(fa[n / 4][n % 4], at_a ^ (n / 4 * 64)); });
            };
            auto read_b = [&](auto part) {
                vl_for<4>([&](auto n) { vl_read<B_AT + (part * 2 + n % 2) * 2048>(fb[part][n / 2][n % 2], at_b ^ (n / 2 * 64)); });
            };
            bf16x8 a_[2][4];
            auto pair = [&](int half, int part, int kk, int i, bool fresh = false) {
                if (fresh) a_[kk][i] = vl_take(fa[kk][i]);
                const bf16x8 a = a_[kk][i];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    f32x4& c = acc[half * 4 + i][part * 2 + j];
                    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b[part][kk][j], a, (FIRST && kk == 0) ? zero4 : c, 0, 0, 0);
                }
            };
            auto falling = [&](int half, int part) {  // A fragments just requested: each pair of MFMAs waits for its own
                vl_wait_lds<7>();
                if (part == 0) {
                    take_b(0, 0);
                    take_b(0, 1);
                }
                pair(half, part, 0, 0, true);
                vl_wait_lds<6>(); pair(half, part, 0, 1, true);
                vl_wait_lds<5>(); pair(half, part, 0, 2, true);
                vl_wait_lds<4>(); pair(half, part, 0, 3, true);
                vl_wait_lds<3>(); pair(half, part, 1, 0, true);
                vl_wait_lds<2>(); pair(half, part, 1, 1, true);
                vl_wait_lds<1>(); pair(half, part, 1, 2, true);
                vl_wait_lds<0>(); pair(half, part, 1, 3, true);
            };
            load(2);
            read_b(C0{});
            read_a(C0{});
            enter();
            falling(0, 0);
            leave();
            load(3);
            read_b(C1{});
            enter();
            vl_wait_lds<2>();
            take_b(1, 0);
#pragma unroll
            for (int i = 0; i < 4; ++i) pair(0, 1, 0, i);
            vl_wait_lds<0>();
            take_b(1, 1);
#pragma unroll
            for (int i = 0; i < 4; ++i) pair(0, 1, 1, i);
            leave();
            load(0);
            read_a(C1{});
            enter();
            falling(1, 1);
            leave();
            load(1);
            enter();
#pragma unroll
            for (int kk = 0; kk < 2; ++kk)
#pragma unroll
                for (int i = 0; i < 4; ++i) pair(1, 0, kk, i);
            leave();
        } else if constexpr (KIND == 1) {
            RowFrag fa[2][4];  // [kk][i]
            TrFrag fb[2][4];   // [slice][j]
            auto read_a = [&](auto half, auto kk) {
                vl_for<4>([&](auto i) { vl_read<(half * 4 + i) * 2048>(fa[kk][i], at_a ^ (kk * 64)); });
            };
            auto read_b = [&](auto kk) {
                vl_for<4>([&](auto j) { vl_read<B_AT + kk * 16384>(fb[kk][j], at_b ^ (j << 5)); });
            };
            bf16x8 a[2][4], b[2][4];
            auto one = [&](int half, int kk, int i, int j) {
                // the first slice a half of the rows meets starts from zero: slice 0 for the lower, slice 1 for the upper rows
                f32x4& c = acc[half * 4 + i][j];
                c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b[kk][j], a[kk][i], (FIRST && kk == half) ? zero4 : c, 0, 0, 0);
            };
            auto row = [&](int half, int kk, int i) {
                a[kk][i] = vl_take(fa[kk][i]);
#pragma unroll
                for (int j = 0; j < 4; ++j) one(half, kk, i, j);
            };
            load(2);
            read_b(C0{});
            read_a(C0{}, C0{});
            read_a(C0{}, C1{});
            enter();
            vl_wait_lds<7>();
#pragma unroll
            for (int j = 0; j < 4; ++j) b[0][j] = vl_take(fb[0][j]);
            row(0, 0, 0);
            vl_wait_lds<6>(); row(0, 0, 1);
            vl_wait_lds<5>(); row(0, 0, 2);
            vl_wait_lds<4>(); row(0, 0, 3);
            leave();
            load(3);
            read_b(C1{});
            enter();
            auto column = [&](int j) {
                b[1][j] = vl_take(fb[1][j]);
#pragma unroll
                for (int i = 0; i < 4; ++i) one(0, 1, i, j);
            };
            vl_wait_lds<6>();
#pragma unroll
            for (int i = 0; i < 4; ++i) a[1][i] = vl_take(fa[1][i]);
            column(0);
            vl_wait_lds<4>(); column(1);
            vl_wait_lds<2>(); column(2);
            vl_wait_lds<0>(); column(3);
            leave();
            load(0);
            read_a(C1{}, C1{});
            read_a(C1{}, C0{});
            enter();
            vl_wait_lds<7>(); row(1, 1, 0);
            vl_wait_lds<6>(); row(1, 1, 1);
            vl_wait_lds<5>(); row(1, 1, 2);
            vl_wait_lds<4>(); row(1, 1, 3);
            leave();
            load(1);
            enter();
            vl_wait_lds<0>();
#pragma unroll
            for (int i = 0; i < 4; ++i) row(1, 0, i);
            leave();
        } else {
            TrFrag fa[2][4], fb[4];  // [alternating][i], [j] of the slice
            bf16x8 b[4];
            auto phase = [&](auto kk_, auto half_) {
                constexpr int kk = decltype(kk_)::value, half = decltype(half_)::value;
                load((kk * 2 + half + 2) & 3);
                if constexpr (half == 0) vl_for<4>([&](auto j) { vl_read<B_AT + kk * 16384>(fb[j], at_b ^ (j << 5)); });
                vl_for<4>([&](auto i) { vl_read<kk * 16384>(fa[half][i], at_a ^ ((half * 4 + i) << 5)); });
                enter();
                auto row = [&](int i) {
                    const bf16x8 a = vl_take(fa[half][i]);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        f32x4& c = acc[half * 4 + i][j];
                        c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b[j], a, (FIRST && kk == 0) ? zero4 : c, 0, 0, 0);
                    }
                };
                vl_wait_lds<6>();
                if constexpr (half == 0) vl_for<4>([&](auto j) { b[j] = vl_take(fb[j]); });
                row(0);
                vl_wait_lds<4>(); row(1);
                vl_wait_lds<2>(); row(2);
                vl_wait_lds<0>(); row(3);
                leave();
            };
            phase(C0{}, C0{});
            phase(C0{}, C1{});
            phase(C1{}, C0{});
            phase(C1{}, C1{});
        }
        at_a ^= STAGE * 2;
        at_b ^= STAGE * 2;
    };

    load_unit(first);
    load(0); load(1); load(2); load(3); load(0); load(1);
    asm volatile("s_waitcnt vmcnt(8)\n\ts_barrier" ::: "memory");
    if (wm == 1) asm volatile("s_barrier" ::: "memory");  // wave row 1 runs one barrier behind row 0 from here on
    for (int u = first; u < units; u += G) {
        const Unit w = unit_of(u);
        step(std::true_type{});
        for (int s = 1; s < w.steps; ++s) step(std::false_type{});
        // both wave rows write their part at the same time: row 0 gives up its lead, row 1 falls back behind it afterwards
        if (wm == 0) asm volatile("s_barrier" ::: "memory");
        // lane: row m = 16 i + (lane & 15), columns n = 16 j + 4 (lane >> 4) + 0 .. 3 of the wave's 128 x 64
        const int mw = w.m0 + wm * 128, nw = w.n0 + wn * 64;
        if (KIND != 0 && w.part >= 0) {
            float* dst = p.part + (static_cast<size_t>(w.part) * 32 * 512 + tid) * 4;
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) *reinterpret_cast<f32x4*>(dst + (i * 4 + j) * 2048) = acc[i][j];
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int m = mw + i * 16 + r16;
                if (mw + i * 16 >= p.M) break;  // (few rows: most of the tile)
                if constexpr (KIND == 0) {
                    if (nw + 64 > p.N) {  // (the last columns of the vocabulary)
#pragma unroll
                        for (int j = 0; j < 4; ++j)
#pragma unroll
                            for (int e = 0; e < 4; ++e) acc[i][j][e] = nw + j * 16 + 4 * g4 + e < p.N ? acc[i][j][e] : -VL_INF;
                    }
                    float mx = acc[i][0][0];
#pragma unroll
                    for (int j = 0; j < 4; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e) mx = fmaxf(mx, acc[i][j][e]);
                    mx = vl_max4(mx) * p.scale_log2;
                    const float ref = mx == -VL_INF ? 0.f : mx;  // (a group beyond the vocabulary, or one that is masked out)
                    float sum = 0.f;
#pragma unroll
                    for (int j = 0; j < 4; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            acc[i][j][e] = vl_exp2(fmaf(acc[i][j][e], p.scale_log2, -ref));
                            sum += acc[i][j][e];
                        }
                    sum = vl_sum4(sum);
                    if (g4 == 0 && m < p.M && nw < p.N) p.stats[static_cast<size_t>(m) * p.groups + (nw >> 6)] = float2{mx, sum};
                    if (p.e == nullptr) continue;
                }
                if (KIND == 0 || p.out != nullptr) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        bf16x4 v;
#pragma unroll
                        for (int e = 0; e < 4; ++e) v[e] = f32_to_bf16(KIND == 0 ? acc[i][j][e] : acc[i][j][e] * alpha);
                        *reinterpret_cast<bf16x4*>(stage + r16 * 64 + (((2 * j + (g4 >> 1)) ^ (r16 & 7)) << 3) + 4 * (g4 & 1)) = v;
                    }
#pragma unroll
                    for (int ps = 0; ps < 2; ++ps) {
                        const int row = ps * 8 + (lane >> 3), ch = lane & 7;
                        const bf16x8 v = *reinterpret_cast<const bf16x8*>(stage + row * 64 + ((ch ^ (row & 7)) << 3));
                        const int mm = mw + i * 16 + row, nn = nw + ch * 8;
                        if (KIND == 0) {
                            if (mm < p.M && nn < p.lde) vl_store(reinterpret_cast<bf16x8*>(p.e + mm * p.lde + nn), v, p.stream);
                        } else {
                            if (mm < p.M && nn < p.N) *reinterpret_cast<bf16x8*>(p.out + mm * p.ldo + nn) = v;
                        }
                    }
                } else if (m < p.M) {
                    float* dst = p.out32 + m * p.ldo + nw + 4 * g4;
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (nw + j * 16 + 4 * g4 < p.N) {
                            f32x4 v;
#pragma unroll
                            for (int e = 0; e < 4; ++e) v[e] = acc[i][j][e] * alpha;
                            f32x4* at = reinterpret_cast<f32x4*>(dst + j * 16);
                            *at = p.accumulate ? *at + v : v;
                        }
                }
            }
        }
        if (wm == 1) asm volatile("s_barrier" ::: "memory");
    }
    if (wm == 0) asm volatile("s_barrier" ::: "memory");  // pairs with the last barrier of wave row 1
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");      // the loader's trailing units
}

// The tiles that were cut along k: their parts summed in order, times alpha.  A workgroup takes 16 rows of both wave rows
// and 16 columns of every wave column, a thread the four values that one thread of the product held.
__global__ __launch_bounds__(512) void vocab_join_kernel(const VocabGemm p) {
    const int t = blockIdx.x >> 5, ij = blockIdx.x & 31, i = ij >> 2, j = ij & 3, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int m0, n0;
    vl_tile(p, p.whole + t, m0, n0);
    const int m = m0 + (wave >> 2) * 128 + i * 16 + (lane & 15), n = n0 + (wave & 3) * 64 + j * 16 + 4 * (lane >> 4);
    if (m >= p.M || n >= p.N) return;
    const float alpha = p.alpha[0];
    const float* src = p.part + ((static_cast<size_t>(t) * p.parts * 32 + ij) * 512 + tid) * 4;
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
    int k = 0;
    for (; k + 8 <= p.parts; k += 8) {
        f32x4 v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = *reinterpret_cast<const f32x4*>(src + static_cast<size_t>(k + e) * 32 * 2048);
#pragma unroll
        for (int e = 0; e < 8; ++e) s += v[e];
    }
    for (; k < p.parts; ++k) s += *reinterpret_cast<const f32x4*>(src + static_cast<size_t>(k) * 32 * 2048);
    if (p.out != nullptr) {
        bf16x4 r;
#pragma unroll
        for (int e = 0; e < 4; ++e) r[e] = f32_to_bf16(s[e] * alpha);
        *reinterpret_cast<bf16x4*>(p.out + m * p.ldo + n) = r;
    } else {
        f32x4* at = reinterpret_cast<f32x4*>(p.out32 + m * p.ldo + n);
        f32x4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = s[e] * alpha;
        *at = p.accumulate ? *at + v : v;
    }
}

// ------------------------------------------------------------------------------------------------
// targets: weights p, base = sum p ln p (- sum p z / tau behind a projection), whether the row has a target
// ------------------------------------------------------------------------------------------------
struct Targets {
    const long long* ids;    // [rows][top]
    const float* teacher;    // [rows][top], or nullptr: one target of weight 1 (labels)
    float* p;                // [rows][top] weights, of repeated ids at their first entry; unused for labels
    float* z;                // [rows][top] scores of the targets, or nullptr (no gradient, or given logits)
    float* base;             // [rows]
    int* valid;              // [rows]
    const bf16 *x, *w;       // behind a projection: [rows][width], [vocab][width]; else nullptr
    bf16* x_used;            // copy of x with zeros in the rows without a target, or nullptr: what such a row holds (NaN, say)
                             // must not meet its zero gradient in the product that gives dW; rows rounded up to 64, zeros behind the last
    int rows, top, width;
    long long vocab;
    float inv_tau;
};

// a + (a of lane ^ LANES) in the lanes whose bit LANES is clear, the same of b in the others
template <int LANES>
__device__ __forceinline__ float vl_halves(float a, float b) {
    const uint32_t x = __builtin_bit_cast(uint32_t, a), y = __builtin_bit_cast(uint32_t, b);
    u32x2 r;
    if constexpr (LANES == 16) r = __builtin_amdgcn_permlane16_swap(x, y, false, false);
    else r = __builtin_amdgcn_permlane32_swap(x, y, false, false);
    const uint32_t lo = r[0], hi = r[1];
    return __builtin_bit_cast(float, lo) + __builtin_bit_cast(float, hi);
}
// sum of s[lane / 8] over the wave: the first three exchanges each halve the values a lane still has to do with
__device__ __forceinline__ float vl_sums8(const float (&s)[8], int lane) {
    float v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = vl_halves<32>(s[i], s[i + 4]);
    const float a = vl_halves<16>(v[0], v[2]), b = vl_halves<16>(v[1], v[3]);
    float r = (lane & 8 ? b : a) + __shfl_xor(lane & 8 ? a : b, 8, 64);
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) r += __shfl_xor(r, o, 64);
    return r;
}

// - p . (x . W[id]) / tau of a row's targets, eight at a time (their rows of W are on their way together): this wave's share,
// targets first, first + 8, ... of every `step`; lane's part of the sum.  The scores themselves are kept for q - p at the
// targets: a student close to its teacher leaves little of that difference, and q from a rounded exponential would be most of
// its error (70 rows of 64 targets, teacher within 0.003 of the student: dx off by 17 % of it, from these scores by 0.2 %).
template <typename P, typename I>
__device__ __forceinline__ float vl_target_scores(const Targets& t, int row, int first, int step, int lane, P p_of, I id_of) {
    const bf16* x = t.x + static_cast<size_t>(row) * t.width;
    float base = 0.f;
    for (int k0 = first; k0 < t.top; k0 += step) {
        const bf16* w[8];
        float pk[8], s[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            s[i] = 0.f;
            pk[i] = k0 + i < t.top ? p_of(k0 + i) : 0.f;
            w[i] = t.w + (pk[i] != 0.f ? id_of(k0 + i) : 0ll) * t.width;
        }
        for (int c = lane * 8; c < t.width; c += 512) {
            const bf16x8 xv = *reinterpret_cast<const bf16x8*>(x + c);
            bf16x8 wv[8];
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (pk[i] != 0.f) wv[i] = *reinterpret_cast<const bf16x8*>(w[i] + c);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (pk[i] == 0.f) continue;  // (not multiplied by 0: what an absent target's row holds does not count)
#pragma unroll
                for (int e = 0; e < 8; ++e) s[i] = fmaf(bf16_to_f32(xv[e]), bf16_to_f32(wv[i][e]), s[i]);
            }
        }
        const float sum = vl_sums8(s, lane);
        if ((lane & 7) == 0) {
            const int k = k0 + (lane >> 3);
            const float p = k < t.top ? p_of(k) : 0.f;
            if (p != 0.f) {
                base -= p * sum * t.inv_tau;
                if (t.z != nullptr) t.z[static_cast<size_t>(row) * t.top + k] = sum;
            }
        }
    }
    return base;
}
__device__ __forceinline__ void vl_copy_used(const Targets& t, int row, int at, int threads, bool some) {
    if (t.x_used == nullptr) return;
    for (int c = at * 8; c < t.width; c += threads * 8) {
        const size_t o = static_cast<size_t>(row) * t.width + c;
        *reinterpret_cast<bf16x8*>(t.x_used + o) = some ? *reinterpret_cast<const bf16x8*>(t.x + o) : bf16x8{};
    }
}

// labels: one wave per row
__global__ __launch_bounds__(256) void vocab_labels_kernel(const Targets t) {
    const int lane = threadIdx.x & 63, row = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= t.rows) {
        vl_copy_used(t, row, lane, 64, false);
        return;
    }
    const long long id = t.ids[row];
    const bool some = id >= 0 && id < t.vocab;
    const float base = wave_sum(some ? vl_target_scores(t, row, 0, 8, lane, [](int) { return 1.f; }, [&](int) { return id; }) : 0.f);
    vl_copy_used(t, row, lane, 64, some);
    if (lane == 0) {
        t.base[row] = base;
        t.valid[row] = some ? 1 : 0;
    }
}

// a teacher: one workgroup per row, of four waves where there are rows of W to fetch (512 rows of 32 targets, width 768: 12 us,
// with one wave 17; 8192 rows of 64 targets, width 1024: 157, 172) or targets by the hundred, else of one (8192 rows of 64
// targets on given logits: 17 us, with four 46).  What is left of an id that repeats is its first entry, with all their weight.
template <int THREADS>
__global__ __launch_bounds__(THREADS) void vocab_teacher_kernel(const Targets t) {
    extern __shared__ __attribute__((aligned(16))) int vl_targets_lds[];
    __shared__ float red[16];
    const int tid = threadIdx.x, row = blockIdx.x, padded = (t.top + 3) & ~3;
    int* id = vl_targets_lds;
    float *p = reinterpret_cast<float*>(id + padded), *merged = p + padded;
    if (row >= t.rows) {
        vl_copy_used(t, row, tid, THREADS, false);
        return;
    }
    const long long* ids = t.ids + static_cast<size_t>(row) * t.top;
    const float* z = t.teacher + static_cast<size_t>(row) * t.top;
    float mx = -VL_INF;
    int any = 0;
    for (int k = tid; k < padded; k += THREADS) {
        const bool ok = k < t.top && ids[k] >= 0 && ids[k] < t.vocab;
        const float v = ok ? z[k] : -VL_INF;
        id[k] = ok ? static_cast<int>(ids[k]) : -1;
        p[k] = v;
        any |= ok && !(v == -VL_INF);  // (NaN counts: it is to be seen in the loss)
        mx = fmaxf(mx, v);
    }
    const bool some = __syncthreads_or(any) != 0;
    mx = block_max(mx, red);
    if (mx == -VL_INF) mx = 0.f;
    float sum = 0.f;
    for (int k = tid; k < t.top; k += THREADS) sum += vl_exp2((p[k] - mx) * t.inv_tau * VL_LOG2E);
    sum = block_sum(sum, red);
    const float ls = log2f(sum), inv = some ? 1.f / sum : 0.f;
    float base = 0.f;
    for (int k = tid; k < padded; k += THREADS) {
        const float l = (p[k] - mx) * t.inv_tau * VL_LOG2E, pk = id[k] >= 0 && some ? vl_exp2(l) * inv : 0.f;
        p[k] = pk;
        if (pk != 0.f) base += pk * (l - ls) * VL_LN2;
    }
    __syncthreads();
    for (int k = tid; k < t.top; k += THREADS) {
        const int mine = id[k];
        float m = 0.f;
        bool first = mine >= 0;
        for (int j = 0; j < padded; j += 4) {
            const int4 i4 = *reinterpret_cast<const int4*>(id + j);
            const float4 p4 = *reinterpret_cast<const float4*>(p + j);
            m += (i4.x == mine ? p4.x : 0.f) + (i4.y == mine ? p4.y : 0.f) + (i4.z == mine ? p4.z : 0.f) + (i4.w == mine ? p4.w : 0.f);
            first &= !((i4.x == mine && j < k) || (i4.y == mine && j + 1 < k) || (i4.z == mine && j + 2 < k) || (i4.w == mine && j + 3 < k));
        }
        m = first ? m : 0.f;
        merged[k] = m;
        t.p[static_cast<size_t>(row) * t.top + k] = m;
    }
    __syncthreads();
    if (t.x != nullptr && some)
        base += vl_target_scores(t, row, 8 * (tid >> 6), THREADS / 8, tid & 63, [&](int k) { return merged[k]; }, [&](int k) { return static_cast<long long>(id[k]); });
    vl_copy_used(t, row, tid, THREADS, some);
    base = block_sum(base, red);
    if (tid == 0) {
        t.base[row] = base;
        t.valid[row] = some ? 1 : 0;
    }
}

// scal[0] = tau / rows with a target (0 without any)
__global__ __launch_bounds__(1024) void vocab_count_kernel(const int* __restrict__ valid, int rows, float tau, float* __restrict__ scal) {
    __shared__ int red[16];
    int c = 0;
    for (int i = threadIdx.x; i < rows; i += 1024) c += valid[i];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) c += __shfl_xor(c, o, 64);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = c;
    __syncthreads();
    if (threadIdx.x == 0) {
        int n = 0;
        for (int i = 0; i < 16; ++i) n += red[i];
        scal[0] = n > 0 ? tau / n : 0.f;
    }
}

__global__ __launch_bounds__(1024) void vocab_mean_kernel(const float* __restrict__ row_loss, const int* __restrict__ valid, int rows, float tau,
                                                         float* __restrict__ loss) {
    __shared__ float red[16];
    float s = 0.f, n = 0.f;  // (fewer than 2^22 rows: counted exactly)
    for (int i = threadIdx.x; i < rows; i += 1024) {
        s += row_loss[i];
        n += valid[i];
    }
    s = block_sum(s, red);
    n = block_sum(n, red);
    if (threadIdx.x == 0) loss[0] = n > 0.f ? s * (tau * tau / n) : 0.f;
}

// ---- behind a projection: one workgroup per row joins the groups; training: exponentials -> q - p in place (e holds rows
// rounded up to 64)
struct Rows {
    const float2* stats;
    bf16* e;
    long long lde;
    const long long* ids;
    const float* p;          // nullptr: labels
    const float* z;          // scores of the targets
    const float* base;
    const int* valid;
    float* row_loss;
    int groups, top, rows;
    long long vocab;
    bool stream;
    float scale_log2;
};

static_assert(VL_MAX_TOP <= 1024, "a thread per target");
// (of 1024 threads: 8192 rows of 50257 entries 285 us for labels, 297 for 64 targets; before the targets' lines were read first 290
// and 314, with 512 threads 297 and 321, with 256 312 and 337.  At 5.5 to 5.8 TB/s it is bound by memory.)
__global__ __launch_bounds__(1024) void vocab_rows_kernel(const Rows a) {
    constexpr int THREADS = 1024;
    __shared__ float red[16];
    const int row = blockIdx.x, tid = threadIdx.x;
    if (row >= a.rows) {  // rows up to a multiple of 64: zeros for the product over the rows
        for (long long c = tid * 8; c < a.lde; c += THREADS * 8) *reinterpret_cast<bf16x8*>(a.e + row * a.lde + c) = bf16x8{};
        return;
    }
    // this thread's target, on its way under the sums (what it holds counts where p is not 0)
    const size_t target = static_cast<size_t>(row) * a.top + tid;
    const bool one = a.e != nullptr && tid < a.top;
    const float p = one ? (a.p == nullptr ? 1.f : a.p[target]) : 0.f, z = one ? a.z[target] : 0.f;
    const int at = one ? static_cast<int>(a.ids[target]) : 0;
    const float2* st = a.stats + static_cast<size_t>(row) * a.groups;
    float m = -VL_INF;
    for (int g = tid; g < a.groups; g += THREADS) m = fmaxf(m, st[g].x);
    m = block_max(m, red);
    const float ref = m == -VL_INF ? 0.f : m;
    float s = 0.f;
    for (int g = tid; g < a.groups; g += THREADS) s += st[g].y * vl_exp2(st[g].x - ref);
    s = block_sum(s, red);
    // (probabilities from differences to the maximum: rounding ref + ls would show in them where exponents are large, at low temperatures)
    const float ls = log2f(s);
    const bool valid = a.valid[row] != 0;
    if (tid == 0) a.row_loss[row] = valid ? a.base[row] + (ref + ls) * VL_LN2 : 0.f;
    if (a.e == nullptr) return;
    bf16* e = a.e + row * a.lde;
    if (!valid) {
        for (long long c = tid * 8; c < a.lde; c += THREADS * 8) *reinterpret_cast<bf16x8*>(e + c) = bf16x8{};
        return;
    }
    // The loop goes around the caches, and a store of two bytes behind it would fetch its line again: the targets' lines are read into
    // them before any thread gets there (the value is of no use; 64 targets a row: 315 -> 297 us, labels 290 -> 285).
    float line = p != 0.f ? bf16_to_f32(e[at]) : 0.f;
    asm volatile("" : "+v"(line));
    __syncthreads();
    for (long long c = tid * 8; c < a.lde; c += THREADS * 8) {
        const float f = vl_exp2(st[c >> 6].x - ref - ls);
        bf16x8 v = __builtin_nontemporal_load(reinterpret_cast<const bf16x8*>(e + c));
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = f32_to_bf16(bf16_to_f32(v[k]) * f);
        vl_store(reinterpret_cast<bf16x8*>(e + c), v, a.stream);
    }
    __syncthreads();  // every entry is rewritten
    if (p != 0.f) e[at] = f32_to_bf16(vl_exp2(fmaf(z, a.scale_log2, -ref) - ls) - p);
}

// ---- on given logits: one workgroup per row
template <typename T>
struct Logits {
    const T* z;
    T* dz;                   // [rows][ldd], or nullptr; entries behind the vocabulary become zeros
    long long ldz, ldd;
    const long long* ids;
    const float* p;
    const float* base;
    const int* valid;
    const float* scal;       // nullptr: every workgroup counts the rows with a target itself
    const int* every;        // valid of all rows
    float* row_loss;
    int top, vocab, rows;
    float tau;
    float scale_log2, inv_tau;
    bool stream;
};

// 16 bytes of a row that may start at any element
template <typename T>
struct ChunkOf {
    static constexpr int W = 16 / sizeof(T);
    typedef T vec __attribute__((ext_vector_type(W)));
    typedef T any __attribute__((ext_vector_type(W), aligned(sizeof(T))));
};

// The row stays in registers (NV chunks of 16 bytes per thread) between its maximum, its sum and the gradient: one read and
// one write of the logits, 4.5 TB/s on 8192 rows of 50257 in bf16 (364 us).  NV = 0: rows too long for that are read again from
// the caches; rows of all lengths done so: 8192 x 8000 119 us instead of 71, 8192 x 50257 561 instead of 377, 2048 x 131000 319
// instead of 253 (2048 x 140000, too long: 340).  Chunks that a thread holds but the row does not fill cost occupancy: with 13 instead
// of 16 of 512 threads bf16 rows of 33000 entries take 251 us instead of 271, of 50257 394 instead of 414, of 53000 the same 371
// (loss and gradient, 8192 rows); with 1024 threads, fp32 or bf16, there is no difference, so they have 16 alone.
template <typename T, int THREADS, int NV>
__global__ __launch_bounds__(THREADS) void logits_distill_kernel(const Logits<T> a) {
    constexpr int W = 16 / sizeof(T);
    __shared__ float red[16];
    const int row = blockIdx.x, tid = threadIdx.x;
    const T* z = a.z + row * a.ldz;
    const bool valid = a.valid[row] != 0;
    T* dz = a.dz == nullptr ? nullptr : a.dz + row * a.ldd;
    const int chunks = (a.vocab + W - 1) / W;
    if (!valid) {
        if (tid == 0) a.row_loss[row] = 0.f;
        if (dz != nullptr)
            for (int c = tid; c < a.ldd; c += THREADS) dz[c] = static_cast<T>(0.f);
        return;
    }
    typedef typename ChunkOf<T>::vec vec;
    auto load = [&](int c) -> vec {
        if ((c + 1) * W <= a.vocab) return *reinterpret_cast<const typename ChunkOf<T>::any*>(z + c * W);
        vec x;
#pragma unroll
        for (int e = 0; e < W; ++e) x[e] = c * W + e < a.vocab ? z[c * W + e] : static_cast<T>(-VL_INF);
        return x;
    };
    vec held[NV > 0 ? NV : 1];
    if constexpr (NV > 0) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (tid + i * THREADS < chunks) held[i] = load(tid + i * THREADS);
    }
    auto each = [&](auto f) {  // f(chunk index, chunk) over this thread's chunks
        if constexpr (NV > 0) {
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if (tid + i * THREADS < chunks) {
                    u32x4 raw = __builtin_bit_cast(u32x4, held[i]);
                    asm volatile("" : "+v"(raw));  // (converted anew in every pass: the converted row would not fit the registers)
                    f(tid + i * THREADS, __builtin_bit_cast(vec, raw));
                }
        } else {
            for (int c = tid; c < chunks; c += THREADS) f(c, load(c));
        }
    };
    const long long* ids = a.ids + static_cast<size_t>(row) * a.top;
    const float* p = a.p + static_cast<size_t>(row) * a.top;
    float m = -VL_INF;
    each([&](int, vec x) {
#pragma unroll
        for (int e = 0; e < W; ++e) m = fmaxf(m, static_cast<float>(x[e]));
    });
    m = block_max(m, red);
    const float ref = m == -VL_INF ? 0.f : m;
    float s = 0.f, t = 0.f;
    each([&](int, vec x) {
#pragma unroll
        for (int e = 0; e < W; ++e) s += vl_exp2((static_cast<float>(x[e]) - ref) * a.scale_log2);
    });
    for (int k = tid; k < a.top; k += THREADS)
        if (p[k] != 0.f) t += p[k] * (static_cast<float>(z[ids[k]]) - ref);
    s = block_sum(s, red);
    t = block_sum(t, red);
    const float ls = log2f(s);
    if (tid == 0) a.row_loss[row] = a.base[row] - t * a.inv_tau + ls * VL_LN2;
    if (dz == nullptr) return;
    float g;
    if (a.scal != nullptr) {
        g = a.scal[0];
    } else {
        float n = 0.f;
        for (int i = tid; i < a.rows; i += THREADS) n += a.every[i];
        g = a.tau / block_sum(n, red);
    }
    auto q_of = [&](float x) { return vl_exp2((x - ref) * a.scale_log2 - ls); };
    each([&](int c, vec x) {  // (rows of dz are padded to whole chunks, on 16-byte boundaries)
        vec r;
#pragma unroll
        for (int e = 0; e < W; ++e) r[e] = static_cast<T>(q_of(static_cast<float>(x[e])) * g);
        if ((c + 1) * W > a.vocab) {
#pragma unroll
            for (int e = 0; e < W; ++e) r[e] = c * W + e < a.vocab ? r[e] : static_cast<T>(0.f);
        }
        vl_store(reinterpret_cast<vec*>(dz + c * W), r, a.stream);
    });
    for (int c = chunks * W + tid; c < a.ldd; c += THREADS) dz[c] = static_cast<T>(0.f);
    __syncthreads();
    for (int k = tid; k < a.top; k += THREADS)
        if (p[k] != 0.f) dz[ids[k]] = static_cast<T>((q_of(static_cast<float>(z[ids[k]])) - p[k]) * g);
}

// Up to two gradients times g[0], in place, unless it is 1 (a loss that is the root of its graph): nothing is touched then, and
// the grid is one round of workgroups so that finding out is short.
struct Gradients {
    void* at[2];
    long long n[2];  // 16-byte vectors
    bool f32[2];
};
__global__ __launch_bounds__(256) void vocab_scale_kernel(const Gradients a, const float* __restrict__ g) {
    const float gv = g[0];
    if (gv == 1.f) return;
    for (int k = 0; k < 2; ++k)
        for (long long i = blockIdx.x * 256ll + threadIdx.x; i < a.n[k]; i += gridDim.x * 256ll) {
            if (a.f32[k]) {
                f32x4* x = static_cast<f32x4*>(a.at[k]) + i;
                f32x4 v = *x;
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] *= gv;
                *x = v;
            } else {
                bf16x8* x = static_cast<bf16x8*>(a.at[k]) + i;
                bf16x8 v = *x;
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = f32_to_bf16(bf16_to_f32(v[e]) * gv);
                *x = v;
            }
        }
}

// ------------------------------------------------------------------------------------------------
// entry points
// ------------------------------------------------------------------------------------------------
template <typename K>
static int vl_grant_lds(K kernel, int bytes, unsigned long long& granted) {
    int dev = 0;
    if (hipError_t e = hipGetDevice(&dev)) return static_cast<int>(e);
    if (dev < 64 && ((granted >> dev) & 1)) return 0;
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == hipSuccess && dev < 64) granted |= 1ull << dev;
    return static_cast<int>(e);
}

static int vl_cus() {
    static int known[64];
    int dev = 0, n = 0;
    if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return 256;
    if (known[dev] > 0) return known[dev];
    if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n <= 0) n = 256;
    return known[dev] = n;
}

// Tiles in whole rounds of the CUs first; the rest in parts of at least eight K-steps that fill the last round, if it would
// be less than 3/4 full.  Loss and gradients with and without: 64 rows of 50257 entries of width 768 103 and 921 us, 512 rows
// 188 and 987, 2048 rows 537 and 1251, 8192 rows of width 1024 2266 and 2602.
static void vl_plan(VocabGemm& g, bool split) {
    g.tiles_m = pdt_cdiv(g.M, 256);
    g.tiles_n = pdt_cdiv(g.N, 256);
    const int tiles = g.tiles_m * g.tiles_n, steps = pdt_cdiv(g.K, 64), cus = vl_cus();
    g.whole = tiles;
    g.left = 0;
    g.parts = g.part_steps = 1;
    const int rest = tiles % cus;
    if (!split || rest == 0 || rest * 4 >= cus * 3) return;
    int parts = cus / rest;
    if (parts > steps / 8) parts = steps / 8;
    if (parts < 2) return;
    g.part_steps = pdt_cdiv(steps, parts);
    g.parts = pdt_cdiv(steps, g.part_steps);
    g.left = rest;
    g.whole = tiles - rest;
}

template <int KIND>
static int vl_launch(const VocabGemm& g, hipStream_t s) {
    static unsigned long long granted;
    constexpr int lds = (2 * 2 * 256 * 64 + 8 * 16 * 64) * 2;
    if (int e = vl_grant_lds(vocab_gemm_kernel<KIND>, lds, granted)) return e;
    const int units = g.whole + g.left * g.parts, cus = vl_cus();
    hipLaunchKernelGGL(vocab_gemm_kernel<KIND>, dim3(units < cus ? units : cus), dim3(512), lds, s, g);
    if (g.left > 0) hipLaunchKernelGGL(vocab_join_kernel, dim3(g.left * 32), dim3(512), 0, s, g);
    return pdt_launch_status();
}

static bool vl_sizes_ok(int rows, int vocab, int width) {
    // byte offsets inside a tile's rows and a whole number of tiles fit 32 bits
    return rows > 0 && rows < VL_MAX_ROWS && vocab > 0 && vocab < (1 << 22) && width > 0 && width <= (1 << 16) && (width % 64) == 0 &&
           static_cast<long long>(pdt_cdiv(rows, 256)) * pdt_cdiv(vocab, 256) < (1ll << 30) &&
           static_cast<long long>(pdt_cdiv(rows, 256)) * pdt_cdiv(width, 256) < (1ll << 30);
}

static int vl_targets(const long long* ids, const float* teacher, float* p, float* z, float* base, int* valid, float* scal, const void* x, const void* w,
                      void* x_used, int rows, int top, int width, int vocab, float tau, hipStream_t s) {
    Targets t = {ids, teacher, p, z, base, valid, static_cast<const bf16*>(x), static_cast<const bf16*>(w), static_cast<bf16*>(x_used), rows, top, width, vocab, 1.f / tau};
    const int all = x_used == nullptr ? rows : pdt_cdiv(rows, 64) * 64;
    const int lds = (top + 3) / 4 * 4 * 12;
    if (teacher != nullptr && (x != nullptr || top > 128)) hipLaunchKernelGGL(vocab_teacher_kernel<256>, dim3(all), dim3(256), lds, s, t);
    else if (teacher != nullptr) hipLaunchKernelGGL(vocab_teacher_kernel<64>, dim3(all), dim3(64), lds, s, t);
    else hipLaunchKernelGGL(vocab_labels_kernel, dim3(pdt_cdiv(all, 4)), dim3(256), 0, s, t);
    if (scal != nullptr) hipLaunchKernelGGL(vocab_count_kernel, dim3(1), dim3(1024), 0, s, valid, rows, tau, scal);
    return pdt_launch_status();
}

static int vl_mean(const float* row_loss, const int* valid, float* loss, int rows, float tau, hipStream_t s) {
    hipLaunchKernelGGL(vocab_mean_kernel, dim3(1), dim3(1024), 0, s, row_loss, valid, rows, tau, loss);
    return pdt_launch_status();
}

// Scratch of one call, carved from one allocation.
struct Scratch {
    char* at;
    size_t used;
    template <typename T>
    T* take(size_t n) {
        T* r = at == nullptr ? nullptr : reinterpret_cast<T*>(at + used);
        used += (n * sizeof(T) + 255) & ~static_cast<size_t>(255);
        return r;
    }
};
struct RowScratch {
    float *p, *base, *scal, *row_loss;
    int* valid;
    RowScratch(Scratch& m, size_t rows, size_t top, bool teacher) {
        p = teacher ? m.take<float>(rows * top) : nullptr;
        base = m.take<float>(rows);
        row_loss = m.take<float>(rows);
        valid = m.take<int>(rows);
        scal = m.take<float>(1);
    }
};
struct HeadScratch {
    RowScratch r;
    float2* stats;
    bf16 *e, *x_used;
    float *z, *part;
    HeadScratch(Scratch& m, int rows, int top, int vocab, int width, int chunk, bool teacher, bool dx, bool dw) : r(m, rows, top, teacher) {
        const size_t groups = pdt_cdiv(vocab, 64);
        stats = m.take<float2>(chunk * groups);
        e = dx || dw ? m.take<bf16>(static_cast<size_t>(pdt_cdiv(chunk, 64)) * 64 * groups * 64) : nullptr;
        z = dx || dw ? m.take<float>(static_cast<size_t>(rows) * top) : nullptr;
        x_used = dw ? m.take<bf16>(static_cast<size_t>(pdt_cdiv(rows, 64)) * 64 * width) : nullptr;
        size_t need = 0;
        for (int k = 0; k < 2; ++k) {  // a whole chunk, and the last one
            const int n = k == 0 ? chunk : rows % chunk;
            if (n == 0) continue;
            VocabGemm g = {};
            g.N = width;
            g.M = n; g.K = vocab;
            if (dx) vl_plan(g, true);
            if (dx && static_cast<size_t>(g.left) * g.parts > need) need = static_cast<size_t>(g.left) * g.parts;
            g.M = vocab; g.K = n;
            if (dw) vl_plan(g, true);
            if (dw && static_cast<size_t>(g.left) * g.parts > need) need = static_cast<size_t>(g.left) * g.parts;
        }
        part = need > 0 ? m.take<float>(need * 65536) : nullptr;
    }
};

static bool vl_head_ok(int rows, int top, int vocab, int width, int chunk) {
    return vl_sizes_ok(rows, vocab, width) && top > 0 && top <= VL_MAX_TOP && chunk > 0 && chunk <= rows && (chunk == rows || (chunk % 256) == 0);
}

// Bytes of scratch that pdt_head_loss needs; rows are worked off `chunk` at a time (all, or a multiple of 256).
PDT_API long long pdt_head_loss_scratch(int rows, int top, int vocab, int width, int chunk, int teacher, int dx, int dw) {
    if (!vl_head_ok(rows, top, vocab, width, chunk)) return -1;
    Scratch m = {nullptr, 0};
    HeadScratch h(m, rows, top, vocab, width, chunk, teacher != 0, dx != 0, dw != 0);
    return static_cast<long long>(m.used);
}

// Mean loss of x [rows][width] behind w [vocab][width] against ids [rows][top] with weights softmax(teacher / tau), or
// against labels (teacher nullptr, top 1, tau 1); with dx [rows][width] bf16 and dw [vocab][width] in bf16 (dw, one chunk
// only) or fp32 (dw32) where given.  All pointers 16-byte aligned.
PDT_API int pdt_head_loss(const void* x, const void* w, const long long* ids, const float* teacher, float* loss, void* dx, void* dw, float* dw32,
                          void* scratch, long long scratch_bytes, int rows, int top, int vocab, int width, int chunk, float tau, void* stream) {
    if (!vl_head_ok(rows, top, vocab, width, chunk) || !(tau > 0.f) || (dw != nullptr && (dw32 != nullptr || chunk != rows))) return -1;
    if (teacher == nullptr && (top != 1 || tau != 1.f)) return -1;
    const bool want_dw = dw != nullptr || dw32 != nullptr, train = dx != nullptr || want_dw;
    Scratch m = {static_cast<char*>(scratch), 0};
    HeadScratch h(m, rows, top, vocab, width, chunk, teacher != nullptr, dx != nullptr, want_dw);
    if (scratch == nullptr || static_cast<long long>(m.used) > scratch_bytes) return -1;
    hipStream_t s = static_cast<hipStream_t>(stream);
    const long long pitch = (vocab + 63ll) / 64 * 64;
    const bool big = 2 * pitch * chunk >= VL_STREAM_BYTES;
    if (int e = vl_targets(ids, teacher, h.r.p, h.z, h.r.base, h.r.valid, train ? h.r.scal : nullptr, x, w, h.x_used, rows, top, width, vocab, tau, s)) return e;
    for (int r0 = 0; r0 < rows; r0 += chunk) {
        const int n = rows - r0 < chunk ? rows - r0 : chunk;
        VocabGemm g = {};
        g.a = static_cast<const bf16*>(x) + static_cast<size_t>(r0) * width;
        g.b = static_cast<const bf16*>(w);
        g.lda = g.ldb = width;
        g.M = n; g.N = vocab; g.K = width;
        g.stats = h.stats;
        g.e = h.e;
        g.lde = pitch;
        g.stream = big;
        g.groups = pdt_cdiv(vocab, 64);
        g.scale_log2 = VL_LOG2E / tau;
        vl_plan(g, false);
        if (int e = vl_launch<0>(g, s)) return e;
        Rows a = {h.stats, h.e, pitch, ids + static_cast<size_t>(r0) * top, h.r.p == nullptr ? nullptr : h.r.p + static_cast<size_t>(r0) * top,
                  h.z == nullptr ? nullptr : h.z + static_cast<size_t>(r0) * top, h.r.base + r0, h.r.valid + r0, h.r.row_loss + r0, g.groups, top, n, vocab, big, g.scale_log2};
        hipLaunchKernelGGL(vocab_rows_kernel, dim3(train ? pdt_cdiv(n, 64) * 64 : n), dim3(1024), 0, s, a);
        g = {};
        g.lda = pitch; g.ldb = width;
        g.N = width;
        g.a = h.e;
        g.alpha = h.r.scal;
        g.ldo = width;
        g.part = h.part;
        if (dx != nullptr) {
            g.b = static_cast<const bf16*>(w);
            g.M = n; g.K = vocab;
            g.out = static_cast<bf16*>(dx) + static_cast<size_t>(r0) * width;
            vl_plan(g, true);
            if (int e = vl_launch<1>(g, s)) return e;
        }
        if (want_dw) {
            g.b = h.x_used + static_cast<size_t>(r0) * width;
            g.M = vocab; g.K = n;
            g.out = static_cast<bf16*>(dw);
            g.out32 = dw32;
            g.accumulate = r0 > 0;
            vl_plan(g, true);
            if (int e = vl_launch<2>(g, s)) return e;
        }
    }
    return vl_mean(h.r.row_loss, h.r.valid, loss, rows, tau, s);
}

template <typename T>
static int distill_launch(const Logits<T>& a, int rows, hipStream_t s) {
    const int chunks = pdt_cdiv(a.vocab, 16 / static_cast<int>(sizeof(T)));
#define PDT_LD(TH, NV) hipLaunchKernelGGL(HIP_KERNEL_NAME(logits_distill_kernel<T, TH, NV>), dim3(rows), dim3(TH), 0, s, a)
    if (chunks <= 256) PDT_LD(256, 1);
    else if (chunks <= 1024) PDT_LD(256, 4);
    else if (chunks <= 4 * 512) PDT_LD(512, 4);
    else if (chunks <= 8 * 512) PDT_LD(512, 8);
    else if (chunks <= 13 * 512) PDT_LD(512, 13);
    else if (chunks <= 16 * 512) PDT_LD(512, 16);
    else if (chunks <= 16 * 1024) PDT_LD(1024, 16);
    else PDT_LD(1024, 0);
#undef PDT_LD
    return pdt_launch_status();
}

PDT_API long long pdt_distill_scratch(int rows, int top) {
    if (rows <= 0 || rows >= VL_MAX_ROWS || top <= 0 || top > VL_MAX_TOP) return -1;
    Scratch m = {nullptr, 0};
    RowScratch r(m, rows, top, true);
    return static_cast<long long>(m.used);
}

// dtype: 0 fp32, 1 bf16 logits.  dz (may be nullptr) has the logits' type and 16-byte aligned rows of pitch ldd that hold whole
// 16-byte chunks; it is written up to the pitch, zeros behind the vocabulary.
PDT_API int pdt_distill(const void* z, void* dz, const long long* ids, const float* teacher, float* loss, void* scratch, long long scratch_bytes, int rows,
                        int vocab, int top, long long ldz, long long ldd, float tau, int dtype, void* stream) {
    if (rows <= 0 || rows >= VL_MAX_ROWS || vocab <= 0 || vocab >= (1 << 24) || top <= 0 || top > VL_MAX_TOP || ldz < 0 || !(tau > 0.f) ||
        (dz != nullptr && (ldd < (vocab + 7) / 8 * 8 || (ldd % 8) != 0)))
        return -1;
    Scratch m = {static_cast<char*>(scratch), 0};
    RowScratch r(m, rows, top, true);
    if (scratch == nullptr || static_cast<long long>(m.used) > scratch_bytes) return -1;
    hipStream_t s = static_cast<hipStream_t>(stream);
    const float it = 1.f / tau, c = VL_LOG2E * it;
    // up to 1024 rows every workgroup counts the ones with a target itself: a launch less
    float* scal = rows > 1024 && dz != nullptr ? r.scal : nullptr;
    if (int e = vl_targets(ids, teacher, r.p, nullptr, r.base, r.valid, scal, nullptr, nullptr, nullptr, rows, top, 0, vocab, tau, s)) return e;
    const bool big = ldd * rows * (dtype == 1 ? 2 : 4) >= VL_STREAM_BYTES;
    const int e = dtype == 1 ? distill_launch(Logits<bf16>{static_cast<const bf16*>(z), static_cast<bf16*>(dz), ldz, ldd, ids, r.p, r.base, r.valid, scal, r.valid, r.row_loss, top, vocab, rows, tau, c, it, big}, rows, s)
                             : distill_launch(Logits<float>{static_cast<const float*>(z), static_cast<float*>(dz), ldz, ldd, ids, r.p, r.base, r.valid, scal, r.valid, r.row_loss, top, vocab, rows, tau, c, it, big}, rows, s);
    return e != 0 ? e : vl_mean(r.row_loss, r.valid, loss, rows, tau, s);
}

// x and y (nullptr: none; bf16, or fp32 where the flag says so; 16-byte aligned, whole 16-byte vectors) times a device scalar, in
// place; nothing is touched where it is 1.
PDT_API int pdt_scale_gradients(void* x, long long nx, int x_f32, void* y, long long ny, int y_f32, const float* g, void* stream) {
    if (nx < 0 || ny < 0 || (nx % (x_f32 != 0 ? 4 : 8)) != 0 || (ny % (y_f32 != 0 ? 4 : 8)) != 0) return -1;
    const Gradients a = {{x, y}, {x == nullptr ? 0 : nx / (x_f32 != 0 ? 4 : 8), y == nullptr ? 0 : ny / (y_f32 != 0 ? 4 : 8)}, {x_f32 != 0, y_f32 != 0}};
    const long long most = a.n[0] > a.n[1] ? a.n[0] : a.n[1], blocks = (most + 255) / 256;
    if (most == 0) return 0;
    hipLaunchKernelGGL(vocab_scale_kernel, dim3(static_cast<unsigned>(blocks < 2048 ? blocks : 2048)), dim3(256), 0, static_cast<hipStream_t>(stream), a, g);
    return pdt_launch_status();
}
