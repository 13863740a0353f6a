// Softmax attention over packed sequences with grouped heads, head dims 64 and 128 (MFMA, gfx950), forward and backward.
//
//   q   : [T, H, D]   bf16   T rows: the tokens of all sequences, one sequence behind the other
//   k, v: [T, Hk, D]  bf16   query head h reads key / value head h / (H / Hk)
//   out : [T, H, D]   bf16   lse, delta: [H, T] fp32, minus log-sum-exp in units of q.k / minus rowsum(dO * O)   rest: [T, H, D] 8 bits, out's rounding
//   spans: [T] {first, end}: the sequence a row belongs to; {0, 0} for a row outside every sequence (its results are 0)
//
//   o_i = sum_j p_ij v_j,  p_ij = exp(scale q_i.k_j - lse_i),  j in [first, i] (causal) or [first, end)
//   dv_j = sum_i p_ij do_i,  ds_ij = p_ij (do_i.v_j - do_i.o_i),  dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_i ds_ij q_i
//
// A workgroup (4 waves) owns 128 consecutive rows of the PACKED axis, whatever sequences they belong to, and streams the
// other side in tiles of 64 rows over the union of its rows' intervals: every row's interval is one contiguous range, so
// the mask is one unsigned comparison against a per-lane pair of bounds, short sequences share tiles instead of padding
// them, and the grid depends on T alone.  The matrix orientation, the LDS images and the LDS-DMA ring are those of the
// fixed-length kernels (attention_tile.h); a head of 128 is two 64-wide panels of the same image.
//
// Rows of different sequences share tiles, and a masked probability of zero times a NaN is NaN.  Instead of cleaning every
// tile, a wave looks at its finished rows once: a row that holds a non-finite value is computed again over its own
// interval only (row_* functions: one row per wave, no matrix instructions), so what one sequence or a later position
// holds never shows in another row.
#include "attention_tile.h"
#include <type_traits>

struct PackedArgs {
    const bf16 *q, *k, *v, *o, *dout;
    bf16 *out, *dq, *dk, *dv;
    uint8_t* rest;        // [T, H, D] e5m2, see rest_place: what rounding took from out, for the backward pass (or nullptr)
    float* lse;           // (both negated: they are what the products' accumulators start from)
    float* delta;
    float* part;          // split dK / dV: [splits][2][T][Hk][D] fp32 partial sums, or nullptr
    const int2* spans;
    const int4* order;    // [nblk] {block of 128 rows, first and end of the rows it streams}, the ones with the most tiles first
    long long q_row, k_row, v_row, o_row, dq_row, dk_row, dv_row;   // elements between rows ...
    long long q_head, k_head, v_head, dq_head, dk_head, dv_head;    // ... and between heads (o, dout, out: o_row, D)
    int T, H, Hk, group;
    int causal, nblk, splits;
    float scale_log2, scale;
    float unscale;        // 1 / scale_log2
};

#define AP_INF __builtin_inff()

// Tiles in LDS per streamed operand of the dQ kernel: three (two on their way while one is read) for heads of 64; two for heads
// of 128, so that two workgroups fit a CU - with three, one wave per SIMD has nothing to cover its softmax.  The forward kernel
// has two of either: four workgroups of 64-wide heads fit a CU.
template <int NP>
constexpr int ap_ring = NP == 1 ? AT_RING : 2;

__device__ __forceinline__ bool ap_finite(float x) { return (__builtin_bit_cast(uint32_t, x) & 0x7f800000u) != 0x7f800000u; }

// keys row i attends to / queries that attend to row i, as [lo, hi); empty for rows outside every sequence
__device__ __forceinline__ int2 ap_keys_of(const PackedArgs& p, int row) {
    int2 s = row < p.T ? p.spans[row] : int2{0, 0};
    if (p.causal) s.y = min(s.y, row + 1);
    return s;
}
__device__ __forceinline__ int2 ap_queries_of(const PackedArgs& p, int row) {
    int2 s = row < p.T ? p.spans[row] : int2{0, 0};
    if (p.causal && s.y > 0) s.x = row;
    return s;
}

// The lane, opaque to the compiler: what is computed from it behind a loop is not computed (and kept in registers) before.
__device__ __forceinline__ int ap_late(int lane) {
    asm volatile("" : "+v"(lane));
    return lane;
}

// Bounds of a wave's intervals.  Neither end of them falls from row to row, so the first and the last row that has one give
// all four (lanes 32 .. 63 repeat the rows of lanes 0 .. 31).  Rows without an interval put no bounds on the mask: whatever
// their lanes compute is dropped.
struct Bounds {
    int lo, hi;          // union
    int max_lo, min_hi;  // beyond these an element-wise mask is not needed
};
__device__ __forceinline__ Bounds wave_bounds(int2 s, int from, int to) {  // [from, to): the block's, known to hold them where offsets do not fall
    const uint32_t some = static_cast<uint32_t>(__ballot(s.y > s.x));
    if (some == 0) return {INT32_MAX, 0, 0, INT32_MAX};
    const int first = __builtin_ctz(some), last = 31 - __builtin_clz(some);
    return {max(__builtin_amdgcn_readlane(s.x, first), from), min(__builtin_amdgcn_readlane(s.y, last), to), __builtin_amdgcn_readlane(s.x, last),
            __builtin_amdgcn_readlane(s.y, first)};
}

// 64 rows from row r0 (clamped to `last`, the last row that any lane wants) of a [*, row] matrix, D / 64 panels.  The
// address is a wave-uniform base and a 32-bit lane offset: running 64-bit addresses per lane cost registers the kernels
// do not have (the host keeps 64 rows below 2^31 bytes).
template <int NP>
__device__ __forceinline__ void ap_tile_issue(const TileDma& d, const bf16* base, long long row, int r0, int last, bf16* tile, int wave) {
    const char* first = reinterpret_cast<const char*>(base + r0 * row);
    const uint32_t pitch = static_cast<uint32_t>(row) * 2u;
    const int limit = last - r0;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const uint32_t off = static_cast<uint32_t>(min(static_cast<int>(d.row[j]), limit)) * pitch + d.off[j] * 2u;
#pragma unroll
        for (int pn = 0; pn < NP; ++pn)
            __builtin_amdgcn_global_load_lds((at_global_cvoid*)(first + 128 * pn + off), (at_lds_void*)(tile + pn * AT_TILE + (2 * wave + j) * 512), 16, 0, 0);
    }
}

// Fragment reads of a tile (attention_tile.h) with everything but the lane's part in the immediate offset: one set of
// eight addresses per tile serves both operands, all panels and halves.
struct TileAt {
    uint32_t row[4], tr[2][2];
};
__device__ __forceinline__ TileAt tile_at(const FragAddr& fa, uint32_t base) {
    TileAt t;
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) t.row[ks] = base + fa.row[ks];
#pragma unroll
    for (int i = 0; i < 4; ++i) t.tr[i >> 1][i & 1] = base + fa.tr[i >> 1][i & 1];
    return t;
}
template <int OFF>
__device__ __forceinline__ void read_rows(RowFrags& f, const uint32_t (&at)[4]) {
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) asm volatile("ds_read_b128 %0, %1 offset:%2" : "=v"(f.v[ks]) : "v"(at[ks]), "n"(OFF) : "memory");
}
template <int OFF>
__device__ __forceinline__ void read_tr(TrFrags& f, const uint32_t (&at)[2]) {
    asm volatile("ds_read_b64_tr_b16 %0, %1 offset:%2" : "=v"(f.lo[0]) : "v"(at[0]), "n"(OFF) : "memory");
    asm volatile("ds_read_b64_tr_b16 %0, %1 offset:%2" : "=v"(f.hi[0]) : "v"(at[1]), "n"(OFF) : "memory");
    asm volatile("ds_read_b64_tr_b16 %0, %1 offset:%2" : "=v"(f.lo[1]) : "v"(at[0]), "n"(OFF + 2048) : "memory");
    asm volatile("ds_read_b64_tr_b16 %0, %1 offset:%2" : "=v"(f.hi[1]) : "v"(at[1]), "n"(OFF + 2048) : "memory");
}
// f(0), f(1), ... with compile-time indexes
template <int N, typename F>
__device__ __forceinline__ void ap_for(F f) {
    if constexpr (N > 0) {
        ap_for<N - 1>(f);
        f(std::integral_constant<int, N - 1>{});
    }
}
using C0 = std::integral_constant<int, 0>;
using C1 = std::integral_constant<int, 1>;

// the values of reads issued by inline assembly, taken over behind the wait: nothing that uses them can move in front of it
__device__ __forceinline__ void taken(RowFrags& f) { asm volatile("" : "+v"(f.v[0]), "+v"(f.v[1]), "+v"(f.v[2]), "+v"(f.v[3])); }
__device__ __forceinline__ void taken(TrFrags& f) { asm volatile("" : "+v"(f.lo[0]), "+v"(f.lo[1]), "+v"(f.hi[0]), "+v"(f.hi[1])); }
__device__ __forceinline__ void taken(f32x4 (&f)[4]) { asm volatile("" : "+v"(f[0]), "+v"(f[1]), "+v"(f[2]), "+v"(f[3])); }

// What rounding to bf16 took from an output, half a step of it (2^-8 of the value) at most, in 8 bits (e5m2) relative to the output's own
// exponent: with out = m 2^e, 0.5 <= |m| < 1, the rest is 2^(e - 9) at most, and times 2^(24 - e) that is 2^15, 29 octaves above
// e5m2's smallest normal number.  So an eighth of the rest is all that is lost, whatever the size of the values.  The bytes of a row
// lie as the dQ kernel's lanes read them: element d at half d / 8 % 2, 8 (d / 16) + d % 8.
template <int NP>
__device__ __forceinline__ int rest_place(int d) { return ((d >> 3) & 1) * (32 * NP) + ((d >> 4) << 3) + (d & 7); }
__device__ __forceinline__ float rest_of(float x) {
    const float out = bf16_to_f32(f32_to_bf16(x));
    const float r = __builtin_amdgcn_ldexpf(x - out, 24 - __builtin_amdgcn_frexp_expf(out));
    return __builtin_amdgcn_fmed3f(r, -57344.f, 57344.f);  // (NaN comes out as a number: its row is computed again)
}
__device__ __forceinline__ float rest_add(float out, float r) { return out + __builtin_amdgcn_ldexpf(r, __builtin_amdgcn_frexp_expf(out) - 24); }
__device__ __forceinline__ uint32_t rest_pack(float a, float b, float c, float d) {
    const int lo = __builtin_amdgcn_cvt_pk_bf8_f32(a, b, 0, false);
    return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_bf8_f32(c, d, lo, true));
}
// sum over four elements of g[e] (o[e] + rest[e])
__device__ __forceinline__ float rest_dot(uint32_t rest, const bf16* g, const bf16* o, float s) {
    const f32x2 a = __builtin_amdgcn_cvt_pk_f32_bf8(static_cast<int>(rest), false), b = __builtin_amdgcn_cvt_pk_f32_bf8(static_cast<int>(rest), true);
    const float r[4] = {a[0], a[1], b[0], b[1]};
#pragma unroll
    for (int e = 0; e < 4; ++e) s = fmaf(bf16_to_f32(g[e]), rest_add(bf16_to_f32(o[e]), r[e]), s);
    return s;
}

// ---- one row by a whole wave, over its own interval only.  64 rows of the other side at a time: a lane forms the products with
// one of them, then the lanes take elements lane, lane + 64 of the sums.  (One document of 16384 rows, 16 heads of 128 on 4,
// the first value NaN and with it every row: 77 ms forward, 7 ms backward, which ends a row whose elements are all NaN.)
template <int NP>
__device__ __forceinline__ float row_dot(const bf16* a, const bf16* b) {
    float s = 0.f;
#pragma unroll 2
    for (int c = 0; c < 64 * NP; c += 8) {
        const bf16x8 x = *reinterpret_cast<const bf16x8*>(a + c), y = *reinterpret_cast<const bf16x8*>(b + c);
#pragma unroll
        for (int e = 0; e < 8; ++e) s = fmaf(bf16_to_f32(x[e]), bf16_to_f32(y[e]), s);
    }
    return s;
}
// acc[e] += sum over the `count` lanes from 0 of w times element lane + 64 e of row (first + lane's number)
template <int NP>
__device__ __forceinline__ void row_add(float (&acc)[NP], float w, int count, const bf16* first, long long pitch, int lane) {
    auto some = [&](int t0, auto n) {
        bf16 x[n][NP];
#pragma unroll
        for (int t = 0; t < n; ++t)
#pragma unroll
            for (int e = 0; e < NP; ++e) x[t][e] = first[(t0 + t) * pitch + lane + 64 * e];
#pragma unroll
        for (int t = 0; t < n; ++t) {
            const float wt = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, w), t0 + t));
#pragma unroll
            for (int e = 0; e < NP; ++e) acc[e] = fmaf(wt, bf16_to_f32(x[t][e]), acc[e]);
        }
    };
    int t = 0;
    for (; t + 8 <= count; t += 8) some(t, std::integral_constant<int, 8>{});
    for (; t < count; ++t) some(t, std::integral_constant<int, 1>{});
}
template <int NP>
__device__ __forceinline__ bool row_is_nan(const float (&acc)[NP]) {  // every element is, and stays so whatever is added
    bool nan = true;
#pragma unroll
    for (int e = 0; e < NP; ++e) nan &= acc[e] != acc[e];
    return __all(nan);
}

template <int NP>
__device__ __forceinline__ void row_forward(const PackedArgs& p, int h, int row, int lane) {
    const int hk = h / p.group;
    const int2 s = ap_keys_of(p, row);
    const bf16 *q = p.q + row * p.q_row + h * p.q_head, *k = p.k + hk * p.k_head, *v = p.v + hk * p.v_head;
    float o[NP], m = -AP_INF, l = 0.f;
#pragma unroll
    for (int e = 0; e < NP; ++e) o[e] = 0.f;
    for (int j0 = s.x; j0 < s.y; j0 += 64) {
        const int count = min(64, s.y - j0);
        const float a = row_dot<NP>(q, k + (j0 + min(lane, count - 1)) * p.k_row) * p.scale_log2;
        const float mn = fmaxf(m, wave_max(lane < count ? a : -AP_INF)), ref = mn == -AP_INF ? 0.f : mn;
        const float alpha = fast_exp2(m - ref), w = lane < count ? fast_exp2(a - ref) : 0.f;
        l = l * alpha + wave_sum(w);
        m = mn;
        if (l != l) break;  // a score is NaN: so is the row
#pragma unroll
        for (int e = 0; e < NP; ++e) o[e] *= alpha;
        if (!row_is_nan<NP>(o)) row_add<NP>(o, w, count, v + j0 * p.v_row, p.v_row, lane);
    }
#pragma unroll
    for (int e = 0; e < NP; ++e) {
        const long long at = row * p.o_row + h * (64 * NP) + lane + 64 * e;
        const float x = o[e] / l;
        const bf16 r = f32_to_bf16(x);
        p.out[at] = r;
        if (p.rest != nullptr)
            p.rest[row * p.o_row + h * (64 * NP) + rest_place<NP>(lane + 64 * e)] = static_cast<uint8_t>(rest_pack(rest_of(x), 0.f, 0.f, 0.f));
    }
    if (lane == 0) p.lse[static_cast<size_t>(h) * p.T + row] = (log2f(l) + m) * -p.unscale;
}

template <int NP>
__device__ __forceinline__ void row_dq(const PackedArgs& p, int h, int row, int lane) {
    const int hk = h / p.group;
    const int2 s = ap_keys_of(p, row);
    const bf16 *q = p.q + row * p.q_row + h * p.q_head, *k = p.k + hk * p.k_head, *v = p.v + hk * p.v_head;
    const bf16* g = p.dout + row * p.o_row + h * (64 * NP);
    const float lse = p.lse[static_cast<size_t>(h) * p.T + row];
    float dq[NP], dl = 0.f;
#pragma unroll
    for (int e = 0; e < NP; ++e) {
        const long long at = row * p.o_row + h * (64 * NP) + lane + 64 * e;
        const int rest = p.rest[row * p.o_row + h * (64 * NP) + rest_place<NP>(lane + 64 * e)];
        dl += bf16_to_f32(g[lane + 64 * e]) * rest_add(bf16_to_f32(p.o[at]), __builtin_amdgcn_cvt_f32_bf8(rest, 0));
        dq[e] = 0.f;
    }
    dl = wave_sum(dl);
    for (int j0 = s.x; j0 < s.y; j0 += 64) {
        const int count = min(64, s.y - j0);
        const long long j = j0 + min(lane, count - 1);
        const float ds = fast_exp2((row_dot<NP>(q, k + j * p.k_row) + lse) * p.scale_log2) * (row_dot<NP>(g, v + j * p.v_row) - dl);
        row_add<NP>(dq, ds, count, k + j0 * p.k_row, p.k_row, lane);
        if (row_is_nan<NP>(dq)) break;
    }
#pragma unroll
    for (int e = 0; e < NP; ++e) p.dq[row * p.dq_row + h * p.dq_head + lane + 64 * e] = f32_to_bf16(dq[e] * p.scale);
}

// dK or dV (IS_V) from heads [h0, h1) of the key's group
template <int NP, bool IS_V>
__device__ __forceinline__ void row_dkv(const PackedArgs& p, int hk, int h0, int h1, int split, int row, int lane) {
    const int2 s = ap_queries_of(p, row);
    const bf16 *k = p.k + row * p.k_row + hk * p.k_head, *v = p.v + row * p.v_row + hk * p.v_head;
    float acc[NP];
#pragma unroll
    for (int e = 0; e < NP; ++e) acc[e] = 0.f;
    for (int h = h0; h < h1; ++h) {
        const bf16 *q = p.q + h * p.q_head, *g = p.dout + h * (64 * NP);
        for (int i0 = s.x; i0 < s.y; i0 += 64) {
            const int count = min(64, s.y - i0);
            const long long i = i0 + min(lane, count - 1);
            const size_t term = static_cast<size_t>(h) * p.T + i;
            float w = fast_exp2((row_dot<NP>(k, q + i * p.q_row) + p.lse[term]) * p.scale_log2);
            if constexpr (!IS_V) w *= row_dot<NP>(v, g + i * p.o_row) + p.delta[term];
            if constexpr (IS_V) row_add<NP>(acc, w, count, g + i0 * p.o_row, p.o_row, lane);
            else row_add<NP>(acc, w, count, q + i0 * p.q_row, p.q_row, lane);
            if (row_is_nan<NP>(acc)) {
                h = h1;
                break;
            }
        }
    }
#pragma unroll
    for (int e = 0; e < NP; ++e) {
        const float x = IS_V ? acc[e] : acc[e] * p.scale;
        const int c = lane + 64 * e;
        if (p.part != nullptr) {
            const size_t one = static_cast<size_t>(p.T) * p.Hk * (64 * NP);
            p.part[(static_cast<size_t>(split) * 2 + IS_V) * one + (static_cast<size_t>(row) * p.Hk + hk) * (64 * NP) + c] = x;
        } else if (IS_V) {
            p.dv[row * p.dv_row + hk * p.dv_head + c] = f32_to_bf16(x);
        } else {
            p.dk[row * p.dk_row + hk * p.dk_head + c] = f32_to_bf16(x);
        }
    }
}

// Scores of 32 streamed rows (register r holds row (r & 3) + 8 (r >> 2), the upper half wave 4 more) that lie outside
// [lo, hi) become -inf.  The interval is a bit mask first: two instructions per score, none of them a comparison.
__device__ __forceinline__ void mask_outside(f32x16& a, int lo, int hi) {
    auto below = [](int x) { return x >= 32 ? 0xffffffffu : (1u << max(x, 0)) - 1u; };
    const uint32_t in = below(hi) & ~below(lo);
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        const uint32_t keep = static_cast<uint32_t>(static_cast<int>(in << (31 - (r & 3) - 8 * (r >> 2))) >> 31);
        const float x = a[r];  // (a bit cast of a vector's element itself reads element 0)
        a[r] = __builtin_bit_cast(float, (__builtin_bit_cast(uint32_t, x) & keep) | (0xff800000u & ~keep));
    }
}

// rows of a wave (bit = row, either half of the wave may report it) that hold a non-finite value
template <int N>
__device__ __forceinline__ uint32_t bad_rows(const f32x16 (&a)[N], bool counts) {
    float z = 0.f;  // any infinity or NaN times zero is NaN, and stays
#pragma unroll
    for (int t = 0; t < N; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e) z = fmaf(a[t][e], 0.f, z);
    const unsigned long long b = __ballot(counts && !ap_finite(z));
    return static_cast<uint32_t>(b) | static_cast<uint32_t>(b >> 32);
}

// (block, head) of a workgroup, heads fastest: consecutive workgroups go to the eight XCDs in turn, so an XCD keeps to a few
// heads (one in eight where the heads are a multiple of eight) whose rows its L2 serves, and every XCD gets blocks of all
// sizes.  The blocks with the most tiles come first (pack_spans_kernel): 16384 rows of documents of 1 to 1024 tokens fill
// the CUs 2.7 times, and in the order of the rows the last round left them a quarter idle.
__device__ __forceinline__ void ap_unit(const PackedArgs& p, int heads, int& blk, int& h, int& from, int& to) {
    const int rank = blockIdx.x / heads;
    h = blockIdx.x - rank * heads;
    const int4 e = p.order[rank];
    blk = e.x;
    from = e.y;
    to = e.z;
}

// Measured: D = 64, 16381 rows of documents of up to 1024, 16 heads, causal: 49 us - 150 MB of q, k, v, out and rest would take
// 30 at the rate of a large copy; vector work (exponentials, the ends of short rows) and the waits of workgroups that live for
// five tiles make up the rest.  D = 128, one document of 16384 rows, 16 heads on 4, causal: 1.08 ms, 1.02 PFLOP/s; matrix pipe and
// vector ALU are busy 52 % and 45 % of the time, at 1.9 GHz.
template <int NP>
__global__ __launch_bounds__(256, NP == 1 ? 4 : 2) void packed_fwd_kernel(const PackedArgs p) {
    constexpr int TILE = NP * AT_TILE, RING = 2;
    extern __shared__ __attribute__((aligned(1024))) bf16 ap_smem[];
    bf16* sK = ap_smem;                // [RING][TILE]
    bf16* sV = ap_smem + RING * TILE;  // [RING][TILE]
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int hi = lane >> 5, lq = lane & 31;
    int blk, h, k_lo, k_hi;
    ap_unit(p, p.H, blk, h, k_lo, k_hi);
    const int hk = h / p.group;
    const int qw0 = blk * AT_BR + 32 * wave, qrow = qw0 + lq;
    bf16x8 qf[4 * NP];  // B operand of S^T
    {
        const bf16* qp = p.q + min(qrow, p.T - 1) * p.q_row + h * p.q_head + 8 * hi;
#pragma unroll
        for (int ks = 0; ks < 4 * NP; ++ks) qf[ks] = *reinterpret_cast<const bf16x8*>(qp + 16 * ks);
    }
    const int2 span = ap_keys_of(p, qrow);
    const int nt = (k_hi - k_lo + AT_T - 1) / AT_T;
    const bf16* kbase = p.k + hk * p.k_head;
    const bf16* vbase = p.v + hk * p.v_head;

    const TileDma dma = tile_dma_setup(wave, lane);
    const FragAddr fa = frag_addr_setup(lane);
    auto issue = [&](int t, int slot) {
        ap_tile_issue<NP>(dma, kbase, p.k_row, k_lo + t * AT_T, k_hi - 1, sK + slot * TILE, wave);
        ap_tile_issue<NP>(dma, vbase, p.v_row, k_lo + t * AT_T, k_hi - 1, sV + slot * TILE, wave);
    };
    asm volatile("" ::: "memory");  // (the rows' own loads first: the counter of loads under way is in order)
    if (nt > 0) issue(0, 0);
    const Bounds wb = wave_bounds(span, k_lo, k_hi);
    const int t_lo = wb.hi > wb.lo ? (wb.lo - k_lo) / AT_T : nt, t_hi = wb.hi > wb.lo ? (wb.hi - k_lo + AT_T - 1) / AT_T : nt;

    f32x16 o[2 * NP];
#pragma unroll
    for (int d = 0; d < 2 * NP; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[d][e] = 0.f;
    float lsum = 0.f;      // this lane's share of the row sum
    float m = -AP_INF;     // running maximum (log2 units) ...
    float ref = 0.f;       // ... and what the exponents are taken about: the maximum, 0 before the first key
    const uint32_t sk_lds = lds_addr(sK);

    int buf = 0;
    auto next_tile = [&](int t) {
        asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
        const int cur = buf;
        buf ^= 1;
        if (t + 1 < nt) issue(t + 1, buf);
        return cur;
    };
    constexpr int PANEL = AT_TILE * 2, V_AT = RING * TILE * 2;  // bytes
    TileAt at;
    auto enter_tile = [&](int t) { at = tile_at(fa, sk_lds + static_cast<uint32_t>(next_tile(t)) * (TILE * 2)); };
    // scores of a half of 32 keys, masked with -inf
    auto scores = [&](f32x16& acc, auto kt) {
        RowFrags kf[NP];
        ap_for<NP>([&](auto pn) { read_rows<pn * PANEL + kt * 4096>(kf[pn], at.row); });
        lds_wait<0>();
#pragma unroll
        for (int pn = 0; pn < NP; ++pn) taken(kf[pn]);
#pragma unroll
        for (int ks = 0; ks < 4 * NP; ++ks)
            acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(frag_rows_get(kf[ks >> 2], ks & 3), qf[ks], ks == 0 ? f32x16{} : acc, 0, 0, 0);
    };
    auto mask = [&](f32x16& acc, int k0, const int kt) {
        if (k0 >= wb.max_lo && k0 + AT_T <= wb.min_hi) return;
        const int first = k0 + 32 * kt + 4 * hi;
        mask_outside(acc, span.x - first, span.y - first);
    };
    auto probs = [&](f32x16& acc) {  // in place; returns the lane's partial row sum
        float sum = 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            acc[r] = fast_exp2(fmaf(acc[r], p.scale_log2, -ref));
            sum += acc[r];
        }
        return sum;
    };
    TrFrags vf[2 * NP];
    auto read_v = [&](auto kt) {
        ap_for<2 * NP>([&](auto d) { read_tr<V_AT + (d >> 1) * PANEL + kt * 4096>(vf[d], at.tr[d & 1]); });
    };
    auto values = [&](const f32x16& acc) {
        const bf16x8 pb0 = pack_half(acc, 0), pb1 = pack_half(acc, 1);
        lds_wait<0>();
#pragma unroll
        for (int d = 0; d < 2 * NP; ++d) taken(vf[d]);
#pragma unroll
        for (int d = 0; d < 2 * NP; ++d) o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(frag_tr_get(vf[d], 0), pb0, o[d], 0, 0, 0);
#pragma unroll
        for (int d = 0; d < 2 * NP; ++d) o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(frag_tr_get(vf[d], 1), pb1, o[d], 0, 0, 0);
    };
    // a half with the maximum taken first and the sums so far rescaled
    auto careful_half = [&](int k0, auto kt) {
        f32x16 acc;
        scores(acc, kt);
        read_v(kt);
        mask(acc, k0, kt);
        float mx = acc[0];
#pragma unroll
        for (int r = 1; r < 16; ++r) mx = fmaxf(mx, acc[r]);
        mx = other_half_max(mx) * p.scale_log2;
        const float m_new = fmaxf(m, mx), next = m_new == -AP_INF ? 0.f : m_new;
        const float alpha = m == -AP_INF ? 0.f : fast_exp2(ref - next);  // (before the row's first key there is nothing to keep)
        m = m_new;
        ref = next;
        lsum = lsum * alpha + probs(acc);
#pragma unroll
        for (int d = 0; d < 2 * NP; ++d)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[d][e] *= alpha;
        values(acc);
        __builtin_amdgcn_sched_barrier(0);
    };
    // Every lane's first key lies in a tile that starts at or before the wave's largest first key: those tiles take the
    // maximum.  The tiles behind them do not - one multiply-add, one exponential and one addition per score - unless a
    // partial sum outgrows 2^30 (the maximum rose by 30 octaves): that half and the rest of its tile are then done carefully.
    // (Two loops, not a branch in one: around a branch the compiler keeps a second copy of the output's registers.)
    for (int t = 0; t < min(t_lo, nt); ++t) next_tile(t);
    int t = t_lo, kt0 = 0;
    bool entered = false;
    while (t < t_hi) {
        do {
            const int k0 = k_lo + t * AT_T;
            if (!entered) enter_tile(t);
            if (kt0 == 0) careful_half(k0, C0{});
            careful_half(k0, C1{});
            entered = false;
            kt0 = 0;
            ++t;
        } while (t < t_hi && k_lo + t * AT_T <= wb.max_lo);
        for (; t < t_hi; ++t) {
            // Two halves of 32 keys.  Heads of 128: S(0) S(1) | softmax(0) | PV(0) | softmax(1) | PV(1), so that the matrix pipe has
            // work while the vector ALU turns scores into probabilities; heads of 64 one after the other, which takes registers
            // for four waves per SIMD instead of three (16381 rows of documents, 16 heads: 47 us instead of 52).
            const int k0 = k_lo + t * AT_T;
            enter_tile(t);
            entered = true;
            auto finish = [&](f32x16& acc, auto kt) {  // false: the maximum rose
                read_v(kt);
                mask(acc, k0, kt);
                const float l = probs(acc);
                kt0 = kt;
                if (__builtin_expect(__any(!(l <= 1073741824.f)), 0)) {
                    lds_wait<0>();  // (the value fragments are read again)
                    return false;
                }
                lsum += l;
                values(acc);
                return true;
            };
            f32x16 acc[NP];
            scores(acc[0], C0{});
            if constexpr (NP == 2) scores(acc[1], C1{});
            if (!finish(acc[0], C0{})) break;
            if constexpr (NP == 1) {
                __builtin_amdgcn_sched_barrier(0);
                scores(acc[0], C1{});
            }
            if (!finish(acc[NP - 1], C1{})) break;
            entered = false;
            kt0 = 0;
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    for (t = max(t_lo, t_hi); t < nt; ++t) next_tile(t);
    asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
    const bool some = span.y > span.x;
    const float lt = other_half_sum(lsum);
    const float inv = 1.f / lt;
    if (some) {
#pragma unroll
        for (int d = 0; d < 2 * NP; ++d)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[d][e] *= inv;
    } else {
#pragma unroll
        for (int d = 0; d < 2 * NP; ++d)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[d][e] = 0.f;
    }
    if (hi == 0 && qrow < p.T) p.lse[static_cast<size_t>(h) * p.T + qrow] = some ? (log2f(lt) + ref) * -p.unscale : 0.f;
    const int el = ap_late(lane);
    bf16* orow0 = p.out + qw0 * p.o_row + h * (64 * NP);
    bf16* so = sK + wave * (32 * AT_D);
#pragma unroll
    for (int pn = 0; pn < NP; ++pn)
        store_rows32(so, o + 2 * pn, 1.f, el, p.T - qw0, [&](int row) { return orow0 + row * p.o_row + 64 * pn; });
    uint32_t bad = bad_rows(o, some);
    if (p.rest != nullptr) {
        // The backward pass takes dout . out as the row term of dS = P (dP - term).  Where few keys share a row P (dP - term) is
        // a small difference, and the rounding of out would be its largest error: the term is formed from out and its rest.
        // A lane holds elements 4 hi .. 4 hi + 3 of every eight; swapped with the other half of the wave it has whole eights,
        // every other one: the half of the row that lane reads again.
        uint8_t* at = p.rest + (qw0 + (el & 31)) * p.o_row + h * (64 * NP) + (el >> 5) * (32 * NP);
        const bool there = qw0 + (el & 31) < p.T;
#pragma unroll
        for (int d = 0; d < 2 * NP; ++d) {
            u32x4 w;
#pragma unroll
            for (int r2 = 0; r2 < 2; ++r2) {
                float x[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = rest_of(o[d][8 * r2 + e]);
                float even = __builtin_bit_cast(float, rest_pack(x[0], x[1], x[2], x[3])), odd = __builtin_bit_cast(float, rest_pack(x[4], x[5], x[6], x[7]));
                swap_rows32(even, odd);
                w[2 * r2] = __builtin_bit_cast(uint32_t, even);
                w[2 * r2 + 1] = __builtin_bit_cast(uint32_t, odd);
            }
            if (there) *reinterpret_cast<u32x4*>(at + 16 * d) = w;
        }
    }
    const unsigned long long bl = __ballot(some && !ap_finite(lt));
    bad |= static_cast<uint32_t>(bl) | static_cast<uint32_t>(bl >> 32);
    if (__builtin_expect(bad != 0, 0)) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the rows just stored are written over
        for (int r = 0; r < 32; ++r)
            if ((bad >> r) & 1) row_forward<NP>(p, h, qw0 + r, el);
    }
}

// dQ, and the row terms that dK / dV start from.  Measured as the forward kernel: D = 64 65 us (218 MB, 43 us at a copy's rate);
// D = 128 1.42 to 1.48 ms, 1.11 to 1.14 PFLOP/s (three products), matrix pipe busy 60 % at 1.85 GHz.
template <int NP>
__global__ __launch_bounds__(256, NP == 1 ? 3 : 2) void packed_dq_kernel(const PackedArgs p) {
    constexpr int TILE = NP * AT_TILE, RING = ap_ring<NP>;
    extern __shared__ __attribute__((aligned(1024))) bf16 ap_smem[];
    bf16* sK = ap_smem;
    bf16* sV = ap_smem + RING * TILE;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int hi = lane >> 5, lq = lane & 31;
    int blk, h, k_lo, k_hi;
    ap_unit(p, p.H, blk, h, k_lo, k_hi);
    const int hk = h / p.group;
    const int qw0 = blk * AT_BR + 32 * wave, qrow = qw0 + lq;
    const int2 span = ap_keys_of(p, qrow);
    const int nt = (k_hi - k_lo + AT_T - 1) / AT_T;
    const bf16* kbase = p.k + hk * p.k_head;
    const bf16* vbase = p.v + hk * p.v_head;
    const TileDma dma = tile_dma_setup(wave, lane);
    const FragAddr fa = frag_addr_setup(lane);
    auto issue = [&](int t, int slot) {
        ap_tile_issue<NP>(dma, kbase, p.k_row, k_lo + t * AT_T, k_hi - 1, sK + slot * TILE, wave);
        ap_tile_issue<NP>(dma, vbase, p.v_row, k_lo + t * AT_T, k_hi - 1, sV + slot * TILE, wave);
    };
    asm volatile("" ::: "memory");  // (the rows' own loads first: the counter of loads under way is in order)
#pragma unroll
    for (int t = 0; t < RING - 1; ++t)
        if (t < nt) issue(t, t);
    const Bounds wb = wave_bounds(span, k_lo, k_hi);
    const int t_lo = wb.hi > wb.lo ? (wb.lo - k_lo) / AT_T : nt, t_hi = wb.hi > wb.lo ? (wb.hi - k_lo + AT_T - 1) / AT_T : nt;
    bf16x8 qf[4 * NP], dof[4 * NP];
    float nl = 0.f, ndl = 0.f;  // minus log-sum-exp (log2 units), minus delta
    {
        const int qc = min(qrow, p.T - 1);
        const bf16* qp = p.q + qc * p.q_row + h * p.q_head + 8 * hi;
        const long long orow = qc * p.o_row + h * (64 * NP) + 8 * hi;
        float dl = 0.f;
#pragma unroll
        for (int ks = 0; ks < 4 * NP; ++ks) {
            qf[ks] = *reinterpret_cast<const bf16x8*>(qp + 16 * ks);
            dof[ks] = *reinterpret_cast<const bf16x8*>(p.dout + orow + 16 * ks);
        }
        const uint8_t* rest = p.rest + qc * p.o_row + h * (64 * NP) + hi * (32 * NP);
#pragma unroll
        for (int j = 0; j < 2 * NP; ++j) {
            const u32x4 rv = *reinterpret_cast<const u32x4*>(rest + 16 * j);
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const bf16x8 ov = *reinterpret_cast<const bf16x8*>(p.o + orow + 16 * (2 * j + k));
                bf16 g[8], o[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    g[e] = dof[2 * j + k][e];
                    o[e] = ov[e];
                }
                dl = rest_dot(rv[2 * k], g, o, dl);
                dl = rest_dot(rv[2 * k + 1], g + 4, o + 4, dl);
            }
        }
        ndl = -other_half_sum(dl);
        const size_t off = static_cast<size_t>(h) * p.T + qc;
        if (hi == 0 && qrow < p.T) p.delta[off] = ndl;
        nl = p.lse[off] * p.scale_log2;
    }
    f32x16 dq[2 * NP];
#pragma unroll
    for (int d = 0; d < 2 * NP; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) dq[d][e] = 0.f;
    const uint32_t sk_lds = lds_addr(sK);
    constexpr int PANEL = AT_TILE * 2, V_AT = RING * TILE * 2;  // bytes

    int buf = 0;
    auto next_tile = [&](int t) {
        if (RING > 2 && t + 1 < nt) asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(4 * NP) : "memory");
        else asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
        if (t + RING - 1 < nt) issue(t + RING - 1, buf == 0 ? RING - 1 : buf - 1);
        const int cur = buf;
        buf = buf == RING - 1 ? 0 : buf + 1;
        return cur;
    };
    for (int t = 0; t < min(t_lo, nt); ++t) next_tile(t);
    for (int t = t_lo; t < t_hi; ++t) {
        const int k0 = k_lo + t * AT_T;
        const int cur = next_tile(t);
        const TileAt at = tile_at(fa, sk_lds + static_cast<uint32_t>(cur) * (TILE * 2));
        const bool masked = k0 < wb.max_lo || k0 + AT_T > wb.min_hi;
        // (a wave's products go in front of the other waves' vector work, s_setprio: 16384 rows of one document, 1527 -> 1475 us;
        // the forward and the dK / dV kernels lose 4 to 8 % by it)
        auto half = [&](auto kt) {
            if (k0 + 32 * kt >= wb.hi || k0 + 32 * kt + 32 <= wb.lo) return;  // no row of the wave reaches it
            f32x16 s, dp;
            // delta is the initial accumulator of dP where the registers allow (16 equal ones, set once), else an addition
#pragma unroll
            for (int e = 0; e < 16; ++e) dp[e] = NP == 1 ? ndl : 0.f;
            {
                RowFrags f[NP];
                ap_for<NP>([&](auto pn) { read_rows<pn * PANEL + kt * 4096>(f[pn], at.row); });
                lds_wait<0>();
#pragma unroll
                for (int pn = 0; pn < NP; ++pn) taken(f[pn]);
                __builtin_amdgcn_s_setprio(1);
#pragma unroll
                for (int ks = 0; ks < 4 * NP; ++ks)
                    s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(frag_rows_get(f[ks >> 2], ks & 3), qf[ks], ks == 0 ? f32x16{} : s, 0, 0, 0);
                // 64-wide heads: issued before the wait below; 128-wide ones as one run of sixteen behind it (long document: 1462 us,
                // 1505 the other way), in front of which the other wave of the SIMD does its vector work
                if constexpr (NP == 1) asm volatile("" : "+v"(s));
                __builtin_amdgcn_s_setprio(0);
                __builtin_amdgcn_sched_barrier(0);
                ap_for<NP>([&](auto pn) { read_rows<V_AT + pn * PANEL + kt * 4096>(f[pn], at.row); });  // (under the products just issued)
                lds_wait<0>();
#pragma unroll
                for (int pn = 0; pn < NP; ++pn) taken(f[pn]);
                __builtin_amdgcn_s_setprio(1);
#pragma unroll
                for (int ks = 0; ks < 4 * NP; ++ks)
                    dp = __builtin_amdgcn_mfma_f32_32x32x16_bf16(frag_rows_get(f[ks >> 2], ks & 3), dof[ks], dp, 0, 0, 0);
                __builtin_amdgcn_s_setprio(0);
            }
            __builtin_amdgcn_sched_barrier(0);
            TrFrags kf[2 * NP];  // on their way during the vector work
            ap_for<2 * NP>([&](auto d) { read_tr<(d >> 1) * PANEL + kt * 4096>(kf[d], at.tr[d & 1]); });
            if (masked) {
                const int first = k0 + 32 * kt + 4 * hi;
                mask_outside(s, span.x - first, span.y - first);
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = fast_exp2(fmaf(s[r], p.scale_log2, nl)) * (NP == 1 ? dp[r] : dp[r] + ndl);
            const bf16x8 ds0 = pack_half(s, 0), ds1 = pack_half(s, 1);
            lds_wait<0>();
#pragma unroll
            for (int d = 0; d < 2 * NP; ++d) taken(kf[d]);
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int d = 0; d < 2 * NP; ++d) dq[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(frag_tr_get(kf[d], 0), ds0, dq[d], 0, 0, 0);
#pragma unroll
            for (int d = 0; d < 2 * NP; ++d) dq[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(frag_tr_get(kf[d], 1), ds1, dq[d], 0, 0, 0);
            __builtin_amdgcn_s_setprio(0);
            __builtin_amdgcn_sched_barrier(0);
        };
        half(C0{});
        half(C1{});
    }
    for (int t = max(t_lo, t_hi); t < nt; ++t) next_tile(t);
    asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
    const bool some = span.y > span.x;
    if (!some) {
#pragma unroll
        for (int d = 0; d < 2 * NP; ++d)
#pragma unroll
            for (int e = 0; e < 16; ++e) dq[d][e] = 0.f;
    }
    const int el = ap_late(lane);
    bf16* drow0 = p.dq + qw0 * p.dq_row + h * p.dq_head;
    bf16* so = sK + wave * (32 * AT_D);
#pragma unroll
    for (int pn = 0; pn < NP; ++pn)
        store_rows32(so, dq + 2 * pn, p.scale, el, p.T - qw0, [&](int row) { return drow0 + row * p.dq_row + 64 * pn; });
    const uint32_t bad = bad_rows(dq, some);
    if (__builtin_expect(bad != 0, 0)) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        for (int r = 0; r < 32; ++r)
            if ((bad >> r) & 1) row_dq<NP>(p, h, qw0 + r, el);
    }
}

// dK or dV (IS_V) of a wave's 32 keys: bf16 rows (through `so`, 4 KB of LDS of the wave's own) or fp32 partial sums
template <int NP, bool IS_V>
__device__ __forceinline__ void dkv_store(const PackedArgs& p, f32x16 (&acc)[2 * NP], bf16* so, int hk, int h0, int h1, int split, int kw0, bool some,
                                          int lane) {
    const float mult = IS_V ? 1.f : p.scale;
    if (!some) {
#pragma unroll
        for (int d = 0; d < 2 * NP; ++d)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[d][e] = 0.f;
    }
    const int el = ap_late(lane);
    if (p.part != nullptr) {
        const size_t one = static_cast<size_t>(p.T) * p.Hk * (64 * NP);
        const int row = kw0 + (el & 31);
        float* dst = p.part + (static_cast<size_t>(split) * 2 + IS_V) * one + (static_cast<size_t>(row) * p.Hk + hk) * (64 * NP) + 4 * (el >> 5);
        if (row < p.T) {
#pragma unroll
            for (int d = 0; d < 2 * NP; ++d)
#pragma unroll
                for (int r4 = 0; r4 < 4; ++r4) {
                    f32x4 a;
#pragma unroll
                    for (int e = 0; e < 4; ++e) a[e] = acc[d][4 * r4 + e] * mult;
                    *reinterpret_cast<f32x4*>(dst + 32 * d + 8 * r4) = a;
                }
        }
    } else {
        const long long pitch = IS_V ? p.dv_row : p.dk_row;
        bf16* row0 = IS_V ? p.dv + kw0 * p.dv_row + hk * p.dv_head : p.dk + kw0 * p.dk_row + hk * p.dk_head;
#pragma unroll
        for (int pn = 0; pn < NP; ++pn) store_rows32(so, acc + 2 * pn, mult, el, p.T - kw0, [&](int row) { return row0 + row * pitch + 64 * pn; });
    }
    const uint32_t bad = bad_rows(acc, some);
    if (__builtin_expect(bad != 0, 0)) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        for (int r = 0; r < 32; ++r)
            if ((bad >> r) & 1) row_dkv<NP, IS_V>(p, hk, h0, h1, split, kw0 + r, el);
    }
}

// dK and dV of 64-wide heads.  Measured as the forward kernel: 74 us (201 MB, 40 us at a copy's rate), 80 with two waves per SIMD,
// more of each operand on its way and the row terms applied behind the products.
__global__ __launch_bounds__(256, 3) void packed_dkv64_kernel(const PackedArgs p) {
    constexpr int NP = 1;
    constexpr int TILE = NP * AT_TILE;
    extern __shared__ __attribute__((aligned(1024))) bf16 ap_smem[];
    bf16* sQ = ap_smem;
    bf16* sDO = ap_smem + AT_RING * TILE;
    __shared__ __attribute__((aligned(1024))) float sRow[AT_RING][4][AT_T];  // per tile: lse, delta, two unused rows (waves 2, 3)
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int hi = lane >> 5, lq = lane & 31;
    int blk, u, q_lo, q_hi;
    ap_unit(p, p.Hk * p.splits, blk, u, q_lo, q_hi);
    const int hk = u / p.splits, split = u - hk * p.splits;
    const int h0 = hk * p.group + split * p.group / p.splits, h1 = hk * p.group + (split + 1) * p.group / p.splits;
    const int kw0 = blk * AT_BR + 32 * wave, key = kw0 + lq;
    const int2 span = ap_queries_of(p, key);
    const int nt1 = (q_hi - q_lo + AT_T - 1) / AT_T;  // tiles of one head; the heads follow each other
    const int nt = nt1 * (h1 - h0);
    bf16x8 kf[4 * NP], vf[4 * NP];
    {
        const int kc = min(key, p.T - 1);
        const bf16* kp = p.k + kc * p.k_row + hk * p.k_head + 8 * hi;
        const bf16* vp = p.v + kc * p.v_row + hk * p.v_head + 8 * hi;
#pragma unroll
        for (int ks = 0; ks < 4 * NP; ++ks) {
            kf[ks] = *reinterpret_cast<const bf16x8*>(kp + 16 * ks);
            vf[ks] = *reinterpret_cast<const bf16x8*>(vp + 16 * ks);
        }
    }
    int is_h = h0, is_t = 0;  // the loader's head and tile
    auto issue = [&](int slot) {
        const int r0 = q_lo + is_t * AT_T;
        const TileDma dma = tile_dma_setup(wave, ap_late(lane));  // (worked out anew: registers are what bounds this kernel's waves)
        ap_tile_issue<NP>(dma, p.q + is_h * p.q_head, p.q_row, r0, q_hi - 1, sQ + slot * TILE, wave);
        ap_tile_issue<NP>(dma, p.dout + is_h * (64 * NP), p.o_row, r0, q_hi - 1, sDO + slot * TILE, wave);
        const float* rows = (wave & 1 ? p.delta : p.lse) + static_cast<size_t>(is_h) * p.T;
        __builtin_amdgcn_global_load_lds((at_global_cvoid*)(rows + min(r0 + lane, q_hi - 1)), (at_lds_void*)&sRow[slot][wave][0], 4, 0, 0);
        if (++is_t == nt1) {
            is_t = 0;
            ++is_h;
        }
    };
    asm volatile("" ::: "memory");  // (the rows' own loads first: the counter of loads under way is in order)
#pragma unroll
    for (int i = 0; i < 2; ++i)
        if (i < nt) issue(i);
    const Bounds wb = wave_bounds(span, q_lo, q_hi);
    const int t_lo = wb.hi > wb.lo ? (wb.lo - q_lo) / AT_T : nt1, t_hi = wb.hi > wb.lo ? (wb.hi - q_lo + AT_T - 1) / AT_T : nt1;
    f32x16 dk[2 * NP], dv[2 * NP];
#pragma unroll
    for (int d = 0; d < 2 * NP; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) dk[d][e] = dv[d][e] = 0.f;
    constexpr int DO_AT = AT_RING * TILE * 2;  // bytes
    const uint32_t sq_lds = lds_addr(sQ), srow_lds = lds_addr(&sRow[0][0][0]);

    int buf = 0, done = 0;
    auto next_tile = [&]() {
        if (done + 1 < nt) asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(4 * NP + 1) : "memory");
        else asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
        if (done + 2 < nt) issue(buf == 0 ? AT_RING - 1 : buf - 1);
        const int cur = buf;
        buf = buf == AT_RING - 1 ? 0 : buf + 1;
        ++done;
        return cur;
    };
    for (int hh = h0; hh < h1; ++hh)
        for (int t = 0; t < nt1; ++t) {
            const int cur = next_tile();
            if (t < t_lo || t >= t_hi) continue;
            const int q0 = q_lo + t * AT_T;
            const TileAt at = tile_at(frag_addr_setup(ap_late(lane)), sq_lds + static_cast<uint32_t>(cur) * (TILE * 2));
            const uint32_t row_tile = srow_lds + static_cast<uint32_t>(cur) * (4 * AT_T * 4) + 16 * hi;
            const bool masked = q0 < wb.max_lo || q0 + AT_T > wb.min_hi;
            auto half = [&](auto qt) {
                if (q0 + 32 * qt >= wb.hi || q0 + 32 * qt + 32 <= wb.lo) return;  // no key of the wave meets it
                // (registers: three waves per SIMD have 168 each, 96 of them hold the sums and the keys' own rows; so the row
                // terms start the products' accumulators, and operands are fetched one after the other)
                f32x16 s, dp;
                f32x4 l2[4], nd[4];
                RowFrags f;
#pragma unroll
                for (int r4 = 0; r4 < 4; ++r4) lds_read_f32x4(l2[r4], row_tile + (32 * qt + 8 * r4) * 4);
                read_rows<qt * 4096>(f, at.row);
                lds_wait<0>();
                taken(l2);
                taken(f);
#pragma unroll
                for (int e = 0; e < 16; ++e) s[e] = l2[e >> 2][e & 3];
#pragma unroll
                for (int ks = 0; ks < 4; ++ks) s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(frag_rows_get(f, ks), kf[ks], s, 0, 0, 0);
                asm volatile("" : "+v"(s));  // (the products are issued before the next operand takes their registers)
#pragma unroll
                for (int r4 = 0; r4 < 4; ++r4) lds_read_f32x4(nd[r4], row_tile + AT_T * 4 + (32 * qt + 8 * r4) * 4);
                read_rows<DO_AT + qt * 4096>(f, at.row);
                lds_wait<0>();
                taken(nd);
                taken(f);
#pragma unroll
                for (int e = 0; e < 16; ++e) dp[e] = nd[e >> 2][e & 3];
#pragma unroll
                for (int ks = 0; ks < 4; ++ks) dp = __builtin_amdgcn_mfma_f32_32x32x16_bf16(frag_rows_get(f, ks), vf[ks], dp, 0, 0, 0);
                asm volatile("" : "+v"(dp));
                TrFrags t2[2];  // dO^T, on its way during the vector work
                ap_for<2>([&](auto d) { read_tr<DO_AT + qt * 4096>(t2[d], at.tr[d]); });
                if (masked) {
                    const int first = q0 + 32 * qt + 4 * hi;
                    mask_outside(s, span.x - first, span.y - first);
                }
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    s[r] = fast_exp2(s[r] * p.scale_log2);
                    dp[r] *= s[r];
                }
                bf16x8 pb[2], dsb[2];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    pb[j] = pack_half(s, j);
                    dsb[j] = pack_half(dp, j);
                }
                lds_wait<0>();
#pragma unroll
                for (int d = 0; d < 2; ++d) taken(t2[d]);
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int d = 0; d < 2; ++d) dv[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(frag_tr_get(t2[d], j), pb[j], dv[d], 0, 0, 0);
                __builtin_amdgcn_sched_barrier(0);
                ap_for<2>([&](auto d) { read_tr<qt * 4096>(t2[d], at.tr[d]); });
                lds_wait<0>();
#pragma unroll
                for (int d = 0; d < 2; ++d) taken(t2[d]);
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int d = 0; d < 2; ++d) dk[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(frag_tr_get(t2[d], j), dsb[j], dk[d], 0, 0, 0);
                __builtin_amdgcn_sched_barrier(0);
            };
            half(C0{});
            half(C1{});
        }
    asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
    dkv_store<1, false>(p, dk, sQ + wave * (32 * AT_D), hk, h0, h1, split, kw0, span.y > span.x, lane);
    dkv_store<1, true>(p, dv, sQ + wave * (32 * AT_D), hk, h0, h1, split, kw0, span.y > span.x, lane);
}

// Heads of 128: dK and dV of 32 keys together with both operands' fragments do not leave two waves per SIMD their
// registers, and one wave per SIMD has nothing to run under its softmax.  So a workgroup has two kinds of waves, one pair per
// 32 keys, which the hardware puts on one SIMD:
//   P waves:  S = Q K^T, P = 2^(S - lse), dV += dO^T P            dS waves:  dP = dO V^T - delta, dS = P dP, dK += Q^T dS
// P goes from the one to the other through LDS in fp32, register for register (the two products have the same layout).  The
// work is a sequence of phases of 32 queries with a barrier each; the dS waves run one phase behind.  Tiles are 64 queries
// (32 KB with dO) in a ring of three: one arriving, one of the P waves, one that the dS waves may still need.
// Measured as the forward kernel: 2.20 to 2.33 ms, 0.94 to 1.0 PFLOP/s (four products), matrix pipe busy 46 to 49 %: a phase takes 2400 cycles of which
// the two waves' products are 1024, the rest is each wave's chain from one product over the vector work to the next.  (Products issued behind the wait for
// the other operands instead of between their reads: 3 % slower; all reads issued first: the same; dS
// waves half a phase out of step with the P waves, their dK products under the P waves' exponentials: 2.49 ms; products in front of
// the other waves' vector work by s_setprio: 2.48 ms.)
__global__ __launch_bounds__(512, 2) void packed_dkv128_kernel(const PackedArgs p) {
    constexpr int TILE = 2 * AT_TILE, PANEL = AT_TILE * 2, DO_AT = AT_RING * TILE * 2;  // elements; bytes
    extern __shared__ __attribute__((aligned(1024))) bf16 ap_smem[];
    bf16* sQ = ap_smem;                    // [AT_RING][TILE]
    bf16* sDO = ap_smem + AT_RING * TILE;  // [AT_RING][TILE]
    float* sP = reinterpret_cast<float*>(ap_smem + 2 * AT_RING * TILE);  // [2][4 pairs][16 registers / 4][64 lanes][4]
    __shared__ __attribute__((aligned(1024))) float sRow[AT_RING][8][AT_T];  // a wave's own row terms: lse (P waves) or delta
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int hi = lane >> 5, lq = lane & 31, pair = wave & 3;
    const bool is_p = wave < 4;
    int blk, u, q_lo, q_hi;
    ap_unit(p, p.Hk * p.splits, blk, u, q_lo, q_hi);
    const int hk = u / p.splits, split = u - hk * p.splits;
    const int h0 = hk * p.group + split * p.group / p.splits, h1 = hk * p.group + (split + 1) * p.group / p.splits;
    const int kw0 = blk * AT_BR + 32 * pair, key = kw0 + lq;
    const int2 span = ap_queries_of(p, key);
    const int nt1 = (q_hi - q_lo + AT_T - 1) / AT_T;  // tiles of one head; the heads follow each other
    const int nt = nt1 * (h1 - h0);
    const FragAddr fa = frag_addr_setup(lane);
    // DMA pieces of eight rows: wave w fetches rows 8w .. 8w + 7 of each of the tile's four panels
    const int d_row = wave * 8 + (lane >> 3);
    const uint32_t d_off = ((lane & 7) ^ at_swz(d_row)) << 3;
    bf16x8 own[8];  // B operand: K^T (P waves) or V^T fragments of this lane's key
    {
        const int kc = min(key, p.T - 1);
        const bf16* src = is_p ? p.k + kc * p.k_row + hk * p.k_head : p.v + kc * p.v_row + hk * p.v_head;
#pragma unroll
        for (int ks = 0; ks < 8; ++ks) own[ks] = *reinterpret_cast<const bf16x8*>(src + 8 * hi + 16 * ks);
    }
    int is_h = h0, is_t = 0;  // the loader's head and tile
    auto issue = [&](int slot) {
        const int r0 = q_lo + is_t * AT_T;
        const uint32_t row = static_cast<uint32_t>(min(d_row, q_hi - 1 - r0));
        auto one = [&](const bf16* base, long long pitch, bf16* tile) {
            const char* first = reinterpret_cast<const char*>(base + r0 * pitch);
            const uint32_t off = row * (static_cast<uint32_t>(pitch) * 2u) + d_off * 2u;
#pragma unroll
            for (int pn = 0; pn < 2; ++pn)
                __builtin_amdgcn_global_load_lds((at_global_cvoid*)(first + 128 * pn + off), (at_lds_void*)(tile + pn * AT_TILE + wave * 512), 16, 0, 0);
        };
        one(p.q + is_h * p.q_head, p.q_row, sQ + slot * TILE);
        one(p.dout + is_h * 128, p.o_row, sDO + slot * TILE);
        const float* rows = (is_p ? p.lse : p.delta) + static_cast<size_t>(is_h) * p.T;
        __builtin_amdgcn_global_load_lds((at_global_cvoid*)(rows + min(r0 + lane, q_hi - 1)), (at_lds_void*)&sRow[slot][wave][0], 4, 0, 0);
        if (++is_t == nt1) {
            is_t = 0;
            ++is_h;
        }
    };
    asm volatile("" ::: "memory");  // (the rows' own loads first: the counter of loads under way is in order)
    if (nt > 0) issue(0);
    if (nt > 1) issue(1);
    const Bounds wb = wave_bounds(span, q_lo, q_hi);
    const uint32_t sq_lds = lds_addr(sQ), srow_lds = lds_addr(&sRow[0][wave][0]) + 16 * hi;
    const uint32_t sp_lds = lds_addr(sP) + pair * 4096 + lane * 16;

    // The loop of one kind of waves.  The rows of Q (P waves) or dO that a phase starts from are read during the phase before
    // it, everything else at its start, so that the reads run under products and vector work.  They are waited for before
    // the phase ends: registers with a read under way must not meet a branch (the compiler may move them there).
    // Phases that no key of the wave meets are worked off like others, all masked: the pair waits for the barrier either way.
    auto run = [&](auto role) {
        constexpr bool IS_P = role == 0;
        constexpr int ROWS_AT = IS_P ? 0 : DO_AT, T_AT = IS_P ? DO_AT : 0;
        f32x16 acc[4];  // dV or dK of the 32 keys
#pragma unroll
        for (int d = 0; d < 4; ++d)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[d][e] = 0.f;
        RowFrags f[2];
        f32x4 rt[4];  // row terms
        auto fetch = [&](int slot, auto half) {
            const uint32_t row_at = srow_lds + static_cast<uint32_t>(slot) * (8 * AT_T * 4);
#pragma unroll
            for (int r4 = 0; r4 < 4; ++r4) lds_read_f32x4(rt[r4], row_at + (32 * half + 8 * r4) * 4);
            const uint32_t base = sq_lds + static_cast<uint32_t>(slot) * (TILE * 2);
            uint32_t at[4];
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) at[ks] = base + fa.row[ks];
            read_rows<ROWS_AT + half * 4096>(f[0], at);
            read_rows<ROWS_AT + PANEL + half * 4096>(f[1], at);
        };
        auto fetched = [&]() {
            lds_wait<0>();
            taken(f[0]);
            taken(f[1]);
            taken(rt);
        };
        // queries [q_lo + 64 t + 32 half, + 32) of the current head, tile in ring slot `slot`; then the rows of half2 in slot2
        auto phase = [&](int t, int slot, auto half, int slot2, auto half2) {
            const uint32_t base = sq_lds + static_cast<uint32_t>(slot) * (TILE * 2);
            f32x16 c;
            f32x4 pr[4];  // P of the other wave
            TrFrags ft[4];
            if constexpr (!IS_P) {
#pragma unroll
                for (int r4 = 0; r4 < 4; ++r4) asm volatile("ds_read_b128 %0, %1 offset:%2" : "=v"(pr[r4]) : "v"(sp_lds), "n"(half * 16384 + r4 * 1024) : "memory");
            }
            {
                uint32_t at[2][2];
#pragma unroll
                for (int i = 0; i < 4; ++i) at[i >> 1][i & 1] = base + fa.tr[i >> 1][i & 1];
                ap_for<4>([&](auto d) { read_tr<T_AT + (d >> 1) * PANEL + half * 4096>(ft[d], at[d & 1]); });
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) c[e] = rt[e >> 2][e & 3];  // (the row term starts the sum)
#pragma unroll
            for (int ks = 0; ks < 8; ++ks) c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(frag_rows_get(f[ks >> 2], ks & 3), own[ks], c, 0, 0, 0);
            asm volatile("" : "+v"(c));  // (issued before any wait below)
            if constexpr (IS_P) {
                const int q0 = q_lo + t * AT_T + 32 * half;
                if (q0 < wb.max_lo || q0 + 32 > wb.min_hi) mask_outside(c, span.x - q0 - 4 * hi, span.y - q0 - 4 * hi);
#pragma unroll
                for (int r = 0; r < 16; ++r) c[r] = fast_exp2(c[r] * p.scale_log2);
#pragma unroll
                for (int r4 = 0; r4 < 4; ++r4) {
                    const f32x4 v = {c[4 * r4], c[4 * r4 + 1], c[4 * r4 + 2], c[4 * r4 + 3]};
                    asm volatile("ds_write_b128 %0, %1 offset:%2" ::"v"(sp_lds), "v"(v), "n"(half * 16384 + r4 * 1024) : "memory");
                }
            }
            lds_wait<IS_P ? 4 : 0>();  // (the four writes of P may be under way until the phase ends)
#pragma unroll
            for (int d = 0; d < 4; ++d) taken(ft[d]);
            if constexpr (!IS_P) {
                taken(pr);
#pragma unroll
                for (int r = 0; r < 16; ++r) c[r] *= pr[r >> 2][r & 3];
            }
            const bf16x8 b0 = pack_half(c, 0), b1 = pack_half(c, 1);
            __builtin_amdgcn_sched_barrier(0);
            fetch(slot2, half2);
#pragma unroll
            for (int d = 0; d < 4; ++d) acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(frag_tr_get(ft[d], 0), b0, acc[d], 0, 0, 0);
#pragma unroll
            for (int d = 0; d < 4; ++d) acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(frag_tr_get(ft[d], 1), b1, acc[d], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
            fetched();
        };
        // Tile n + 1 has landed by the second phase of tile n, in which tile n + 2 is requested (into the slot of tile n - 1,
        // which nobody reads any more).
        auto middle = [&](int n, int slot) {
            asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
            if (n + 2 < nt) issue(slot == 0 ? AT_RING - 1 : slot - 1);
        };
        if (nt > 0) {
            if (nt > 1) asm volatile("s_waitcnt vmcnt(5)\n\ts_barrier" ::: "memory");
            else asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
            fetch(0, C0{});
            fetched();
            int slot = 0, t = 0;
            if constexpr (IS_P) {
                for (int n = 0; n < nt; ++n) {
                    const int next = slot == AT_RING - 1 ? 0 : slot + 1;
                    phase(t, slot, C0{}, slot, C1{});
                    middle(n, slot);
                    phase(t, slot, C1{}, n + 1 < nt ? next : slot, C0{});
                    asm volatile("s_barrier" ::: "memory");
                    slot = next;
                    if (++t == nt1) t = 0;
                }
            } else {
                middle(0, 0);
                phase(0, 0, C0{}, 0, C1{});
                asm volatile("s_barrier" ::: "memory");
                for (int n = 1; n < nt; ++n) {
                    const int next = slot == AT_RING - 1 ? 0 : slot + 1;
                    phase(0, slot, C1{}, next, C0{});
                    slot = next;
                    middle(n, slot);
                    phase(0, slot, C0{}, slot, C1{});
                    asm volatile("s_barrier" ::: "memory");
                }
                phase(0, slot, C1{}, slot, C0{});
            }
        }
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        dkv_store<2, IS_P>(p, acc, sQ + wave * (32 * AT_D), hk, h0, h1, split, kw0, span.y > span.x, lane);
    };
    if (is_p) run(C0{});
    else run(C1{});
}

// dK, dV = the sum of the splits' parts, in order
__global__ __launch_bounds__(256) void packed_join_kernel(const PackedArgs p, int D) {
    const long long one = static_cast<long long>(p.T) * p.Hk * D;
    for (long long i = (blockIdx.x * 256ll + threadIdx.x) * 4; i < 2 * one; i += gridDim.x * 1024ll) {
        const bool is_v = i >= one;
        const long long at = is_v ? i - one : i;
        f32x4 a = {0.f, 0.f, 0.f, 0.f};
        for (int s = 0; s < p.splits; ++s) a += *reinterpret_cast<const f32x4*>(p.part + s * 2 * one + i);
        const long long row = at / (p.Hk * D);
        const int rest = static_cast<int>(at - row * (p.Hk * D)), hk = rest / D, d = rest - hk * D;
        bf16x4 r;
#pragma unroll
        for (int e = 0; e < 4; ++e) r[e] = f32_to_bf16(a[e]);
        *reinterpret_cast<bf16x4*>(is_v ? p.dv + row * p.dv_row + hk * p.dv_head + d : p.dk + row * p.dk_row + hk * p.dk_head + d) = r;
    }
}

// Sequence of a row: offsets[s] <= row < offsets[s + 1], cut to the rows there are.  The last sequence that starts at or
// before the row is the only one that can hold it (empty sequences share their start with the one behind them).
template <typename At>
__device__ __forceinline__ int2 pack_span_of(At offset, int n, int rows, int row) {
    int lo = 0, hi = n;  // offsets 0 .. lo - 1 start at or before the row
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (offset(mid) <= row) lo = mid + 1;
        else hi = mid;
    }
    if (lo > 0) {
        const int first = max(offset(lo - 1), 0), end = min(offset(lo), rows);
        if (row < end) return {first, end};
    }
    return {0, 0};
}

// {block of 128 rows, first and end of the rows it streams, their number}: causal query side, causal key side, not causal
template <typename At>
__device__ __forceinline__ int4 pack_entry(At offset, int n, int rows, int b, int kind) {
    const int row = b * AT_BR, last = min(row + AT_BR, rows) - 1;
    const int2 s = pack_span_of(offset, n, rows, row), e = pack_span_of(offset, n, rows, last);
    const int from = kind == 1 || s.y == 0 ? row : s.x, to = kind == 0 || e.y == 0 ? last + 1 : e.y;  // (a block's edge may lie outside every sequence)
    return {b, from, to, to - from};
}

// blocks whose work comes before that of block b: more of it, or as much and in front (w[j]: work of block j0 + j, -1 behind the last)
__device__ __forceinline__ int pack_rank(const int* w, int count, int mine, int before) {
    int rank = 0;
#pragma unroll 16
    for (int j = 0; j < count; j += 4) {
        const int4 x = *reinterpret_cast<const int4*>(w + j);
        rank += (x.x >= mine + (j >= before)) + (x.y >= mine + (j + 1 >= before)) + (x.z >= mine + (j + 2 >= before)) + (x.w >= mine + (j + 3 >= before));
    }
    return rank;
}

// Packs of few blocks and of very many (the last round does not matter, the counting does) keep the rows' own order.  Pack, forward
// and backward in order of falling work and in the rows' own, from a graph: documents of 1 to 4096 rows, 16 heads of 64, 24 blocks
// 123 and 123 us, 32 blocks 148 and 151, 48 210 and 229, 64 300 and 312, 128 304 and 358, 256 790 and 836; 32 heads of 128 on eight,
// 24 blocks 243 and 242, 32 blocks 282 and 302, 64 867 and 864; 4 heads of 64, 32 blocks 138 and 138, 128 182 and 189.  One document
// (ordered either way): within 1 %.  4096 blocks, 2 heads of 64 1202 and 1213, 8192 blocks 2690 and 2385.
#define AP_ORDER_FROM 31
#define AP_ORDER_TO 4096
#define AP_ORDER_ONCE 512    // blocks that one workgroup puts in order, in the launch that makes the spans
#define AP_OFFSETS_LDS 2048  // offsets that are searched in LDS
enum { AP_OWN_ORDER, AP_ORDERED, AP_TO_BE_ORDERED };

// Spans and positions of the rows, a row per thread, and the blocks' entries: in the rows' own order (on the causal query side the
// last blocks first: of a long sequence they have the most keys); by three workgroups in front of the others in the order of
// falling work; or by block, for pack_order_kernel.
__global__ __launch_bounds__(256) void pack_spans_kernel(const int* __restrict__ offsets, int n, int rows, int2* __restrict__ spans,
                                                        long long* __restrict__ positions, int4* __restrict__ entries, int mode) {
    __shared__ int off[AP_OFFSETS_LDS];
    __shared__ __attribute__((aligned(16))) int w[AP_ORDER_ONCE];
    const bool near = n < AP_OFFSETS_LDS;
    if (near) {
        for (int i = threadIdx.x; i <= n; i += 256) off[i] = offsets[i];
        __syncthreads();
    }
    auto offset = [&](int i) { return near ? off[i] : offsets[i]; };
    const int blocks = (rows + AT_BR - 1) / AT_BR, front = mode == AP_ORDERED ? 3 : 0;
    if (static_cast<int>(blockIdx.x) < front) {
        const int kind = blockIdx.x;
        int4 e[AP_ORDER_ONCE / 256];
#pragma unroll
        for (int i = 0; i < AP_ORDER_ONCE / 256; ++i) {
            const int b = threadIdx.x + 256 * i;
            e[i] = b < blocks ? pack_entry(offset, n, rows, b, kind) : int4{0, 0, 0, -1};
            w[b] = e[i].w;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < AP_ORDER_ONCE / 256; ++i) {
            const int b = threadIdx.x + 256 * i;
            if (b < blocks) entries[static_cast<size_t>(kind) * blocks + pack_rank(w, (blocks + 3) & ~3, e[i].w, b)] = e[i];
        }
        return;
    }
    const int row = (blockIdx.x - front) * 256 + threadIdx.x;
    if (row >= rows) return;
    const int2 s = pack_span_of(offset, n, rows, row);
    spans[row] = s;
    positions[row] = s.y > 0 ? row - s.x : 0;
    if (mode != AP_ORDERED && row % AT_BR == 0) {
        const int b = row / AT_BR;
        entries[mode == AP_OWN_ORDER ? blocks - 1 - b : b] = pack_entry(offset, n, rows, b, 0);
        entries[blocks + b] = pack_entry(offset, n, rows, b, 1);
        entries[2 * static_cast<size_t>(blocks) + b] = pack_entry(offset, n, rows, b, 2);
    }
}

// The entries by falling work (equal ones as the rows go).  Counted, not sorted: a few thousand blocks at most.
__global__ __launch_bounds__(256) void pack_order_kernel(const int4* __restrict__ entries, int blocks, int4* __restrict__ order) {
    __shared__ __attribute__((aligned(16))) int w[256];
    const int4* src = entries + static_cast<size_t>(blockIdx.y) * blocks;
    const int b = blockIdx.x * 256 + threadIdx.x;
    const int4 e = b < blocks ? src[b] : int4{0, 0, 0, 0};
    int rank = 0;
    for (int j0 = 0; j0 < blocks; j0 += 256) {
        __syncthreads();
        w[threadIdx.x] = j0 + static_cast<int>(threadIdx.x) < blocks ? src[j0 + threadIdx.x].w : -1;
        __syncthreads();
        rank += pack_rank(w, 256, e.w, b - j0);
    }
    if (b < blocks) order[static_cast<size_t>(blockIdx.y) * blocks + rank] = e;
}

// offsets: [sequences + 1] int32, not falling.  order: [3][ceil(rows / 128)] entries of 16 bytes; work: scratch of the same size.
PDT_API int pdt_pack_spans(const int* offsets, int sequences, int rows, void* spans, long long* positions, void* order, void* work, void* stream) {
    if (sequences < 0 || rows <= 0 || rows >= (1 << 30)) return -1;
    hipStream_t s = static_cast<hipStream_t>(stream);
    const int blocks = pdt_cdiv(rows, AT_BR);
    const int mode = blocks <= AP_ORDER_FROM || blocks > AP_ORDER_TO ? AP_OWN_ORDER : blocks <= AP_ORDER_ONCE ? AP_ORDERED : AP_TO_BE_ORDERED;
    hipLaunchKernelGGL(pack_spans_kernel, dim3(pdt_cdiv(rows, 256) + (mode == AP_ORDERED ? 3 : 0)), dim3(256), 0, s, offsets, sequences, rows,
                       static_cast<int2*>(spans), positions, static_cast<int4*>(mode == AP_TO_BE_ORDERED ? work : order), mode);
    if (mode == AP_TO_BE_ORDERED)
        hipLaunchKernelGGL(pack_order_kernel, dim3(pdt_cdiv(blocks, 256), 3), dim3(256), 0, s, static_cast<const int4*>(work), blocks, static_cast<int4*>(order));
    return pdt_launch_status();
}

static bool ap_stride_ok(const long long* st, int n) {
    for (int i = 0; i < n; ++i)
        if (st[i] <= 0 || (st[i] % 8) != 0 || (i % 2 == 0 && st[i] >= (1 << 24))) return false;
    return true;
}

static int ap_args(PackedArgs& a, const void* spans, const void* order, int T, int H, int Hk, int D, float scale, int causal) {
    if (T <= 0 || H <= 0 || Hk <= 0 || H % Hk != 0 || (D != 64 && D != 128) || !(scale > 0.f) || !(scale < 3.0e38f)) return -1;
    a.spans = static_cast<const int2*>(spans);
    a.T = T; a.H = H; a.Hk = Hk;
    a.group = H / Hk;
    a.nblk = pdt_cdiv(T, AT_BR);
    a.causal = causal != 0;
    a.splits = 1;
    a.order = static_cast<const int4*>(order) + (causal != 0 ? 0 : 2 * static_cast<size_t>(a.nblk));
    a.scale = scale;
    a.scale_log2 = scale * 1.4426950408889634f;
    a.unscale = 1.f / a.scale_log2;
    if (static_cast<long long>(a.nblk) * H >= (1ll << 31) || T >= (1 << 30)) return -1;
    // (out's rows, [H, D] without gaps: as the other strides, see ap_stride_ok.  Inputs whose rows overlap may have shorter ones.)
    if (static_cast<long long>(H) * D >= (1 << 24)) return -1;
    return 0;
}

// Dynamic LDS beyond the default limit is granted once per kernel and device.
template <typename K>
static int ap_lds(K kernel, size_t bytes, unsigned long long& granted) {
    if (bytes <= 64 * 1024) return 0;
    int dev = 0;
    if (hipError_t e = hipGetDevice(&dev)) return static_cast<int>(e);
    if (dev < 64 && ((granted >> dev) & 1)) return 0;
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
    if (e == hipSuccess && dev < 64) granted |= 1ull << dev;
    return static_cast<int>(e);
}

template <typename K>
static int ap_launch(K kernel, unsigned long long& granted, unsigned grid, size_t lds, hipStream_t stream, const PackedArgs& a, int threads = 256) {
    if (int e = ap_lds(kernel, lds, granted)) return e;
    hipLaunchKernelGGL(kernel, dim3(grid), dim3(threads), lds, stream, a);
    return pdt_launch_status();
}

// spans, order: pdt_pack_spans.  st: row and head strides of q, k, v in elements (multiples of 8; 16-byte aligned pointers); out is [T, H, D] without gaps,
// rest (nullptr without a backward pass) has one byte for each of its elements.
PDT_API int pdt_packed_attention_fwd(const void* q, const void* k, const void* v, void* out, void* rest, float* lse, const void* spans, const void* order, const long long* st,
                                     int T, int H, int Hk, int D, float scale, int causal, void* stream) {
    PackedArgs a = {};
    if (ap_args(a, spans, order, T, H, Hk, D, scale, causal) != 0 || !ap_stride_ok(st, 6)) return -1;
    a.q = static_cast<const bf16*>(q);
    a.k = static_cast<const bf16*>(k);
    a.v = static_cast<const bf16*>(v);
    a.out = static_cast<bf16*>(out);
    a.rest = static_cast<uint8_t*>(rest);
    a.lse = lse;
    a.q_row = st[0]; a.q_head = st[1];
    a.k_row = st[2]; a.k_head = st[3];
    a.v_row = st[4]; a.v_head = st[5];
    a.o_row = static_cast<long long>(H) * D;
    const size_t lds = static_cast<size_t>(2 * 2) * AT_T * D * sizeof(bf16);
    const unsigned grid = static_cast<unsigned>(a.nblk) * H;
    static unsigned long long granted[2];
    return D == 64 ? ap_launch(packed_fwd_kernel<1>, granted[0], grid, lds, static_cast<hipStream_t>(stream), a)
                   : ap_launch(packed_fwd_kernel<2>, granted[1], grid, lds, static_cast<hipStream_t>(stream), a);
}

// How many ways the backward pass splits the query heads of a key head (1: no partial sums).  A key block with all the
// heads of its group is one workgroup; with few key heads that leaves CUs idle.  Forward and backward with and without: 4096
// rows, 16 heads of 128 on one key head 333 and 1601 us, 32 on eight 476 and 599 (with up to 1024 workgroups 490); 1024 rows, 16
// heads of 64 on four 80 and 132.
PDT_API int pdt_packed_attention_splits(int T, int H, int Hk) {
    const int group = H / Hk, units = pdt_cdiv(T, AT_BR) * Hk;
    int s = 1;
    while (s < group && units * s < 512) s *= 2;
    return s < group ? s : group;
}

// st: row and head strides of q, k, v, dq, dk, dv; o and dout are [T, H, D] without gaps.  delta: scratch, H * T floats.
// part: scratch, splits * 2 * T * Hk * D floats, unused (may be nullptr) where splits is 1.
PDT_API int pdt_packed_attention_bwd(const void* q, const void* k, const void* v, const void* o, const void* rest, const void* dout, const float* lse, float* delta,
                                     void* dq, void* dk, void* dv, float* part, int splits, const void* spans, const void* order, const long long* st, int T, int H,
                                     int Hk, int D, float scale, int causal, void* stream) {
    PackedArgs a = {};
    if (ap_args(a, spans, order, T, H, Hk, D, scale, causal) != 0 || !ap_stride_ok(st, 12)) return -1;
    if (splits < 1 || splits > a.group || (splits > 1 && part == nullptr) || static_cast<long long>(a.nblk) * Hk * splits >= (1ll << 31)) return -1;
    a.q = static_cast<const bf16*>(q);
    a.k = static_cast<const bf16*>(k);
    a.v = static_cast<const bf16*>(v);
    a.o = static_cast<const bf16*>(o);
    a.rest = const_cast<uint8_t*>(static_cast<const uint8_t*>(rest));
    a.dout = static_cast<const bf16*>(dout);
    a.lse = const_cast<float*>(lse);
    a.delta = delta;
    a.dq = static_cast<bf16*>(dq);
    a.dk = static_cast<bf16*>(dk);
    a.dv = static_cast<bf16*>(dv);
    a.splits = splits;
    a.part = splits > 1 ? part : nullptr;
    a.q_row = st[0]; a.q_head = st[1];
    a.k_row = st[2]; a.k_head = st[3];
    a.v_row = st[4]; a.v_head = st[5];
    a.dq_row = st[6]; a.dq_head = st[7];
    a.dk_row = st[8]; a.dk_head = st[9];
    a.dv_row = st[10]; a.dv_head = st[11];
    a.o_row = static_cast<long long>(H) * D;
    hipStream_t s = static_cast<hipStream_t>(stream);
    const size_t lds = static_cast<size_t>(2 * (D == 64 ? ap_ring<1> : ap_ring<2>)) * AT_T * D * sizeof(bf16);
    const size_t lds_k = static_cast<size_t>(2 * AT_RING) * AT_T * D * sizeof(bf16) + (D == 128 ? 2 * 4 * 4096 : 0);
    const unsigned gq = static_cast<unsigned>(a.nblk) * H, gk = static_cast<unsigned>(a.nblk) * Hk * splits;
    static unsigned long long granted[4];
    int rc = D == 64 ? ap_launch(packed_dq_kernel<1>, granted[0], gq, lds, s, a) : ap_launch(packed_dq_kernel<2>, granted[1], gq, lds, s, a);
    if (a.causal) a.order += a.nblk;  // the key side
    if (rc == 0) rc = D == 64 ? ap_launch(packed_dkv64_kernel, granted[2], gk, lds_k, s, a) : ap_launch(packed_dkv128_kernel, granted[3], gk, lds_k, s, a, 512);
    if (rc != 0) return rc;
    if (a.part != nullptr) {
        const long long n = 2ll * T * Hk * D / 4;
        hipLaunchKernelGGL(packed_join_kernel, dim3(static_cast<unsigned>(n / 256 + 1 < 4096 ? n / 256 + 1 : 4096)), dim3(256), 0, s, a, D);
    }
    return pdt_launch_status();
}
