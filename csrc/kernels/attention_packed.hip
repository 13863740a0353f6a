// Softmax attention over packed sequences with grouped heads, head dims 64 and 128 (MFMA, gfx950), forward and backward.
//
//   q   : [T, H, D]   bf16   T rows: the tokens of all sequences, one sequence behind the other
//   k, v: [T, Hk, D]  bf16   query head h reads key / value head h / (H / Hk)
//   out : [T, H, D]   bf16   lse, delta: [H, T] fp32 (log2 units / minus rowsum(dO * O))
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

struct PackedArgs {
    const bf16 *q, *k, *v, *o, *dout;
    bf16 *out, *dq, *dk, *dv;
    float* lse;
    float* delta;
    float* part;          // split dK / dV: [splits][2][T][Hk][D] fp32 partial sums, or nullptr
    const int2* spans;
    long long q_row, k_row, v_row, o_row, dq_row, dk_row, dv_row;   // elements between rows ...
    long long q_head, k_head, v_head, dq_head, dk_head, dv_head;    // ... and between heads (o, dout, out: o_row, D)
    int T, H, Hk, group;
    int causal, nblk, splits;
    float scale_log2, scale;
};

#define AP_INF __builtin_inff()

// Tiles in LDS per streamed operand of the query-side kernels: three (two on their way while one is read) for heads of 64;
// two for heads of 128, so that two workgroups fit a CU - with three, one wave per SIMD has nothing to cover its softmax.
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

// bounds of a wave's / workgroup's intervals
struct Bounds {
    int lo, hi;          // union
    int max_lo, min_hi;  // beyond these an element-wise mask is not needed
};
__device__ __forceinline__ int wave_min_i(int v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = min(v, __shfl_xor(v, o, 64));
    return v;
}
__device__ __forceinline__ int wave_max_i(int v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = max(v, __shfl_xor(v, o, 64));
    return v;
}
// (rows without an interval put no bounds on the mask: whatever their lanes compute is dropped)
__device__ __forceinline__ Bounds wave_bounds(int2 s) {
    const bool some = s.y > s.x;
    Bounds b;
    b.lo = __builtin_amdgcn_readfirstlane(wave_min_i(some ? s.x : INT32_MAX));
    b.hi = __builtin_amdgcn_readfirstlane(wave_max_i(some ? s.y : 0));
    b.max_lo = __builtin_amdgcn_readfirstlane(wave_max_i(some ? s.x : 0));
    b.min_hi = __builtin_amdgcn_readfirstlane(wave_min_i(some ? s.y : INT32_MAX));
    return b;
}

// 64 rows from row r0 (clamped to `last`, the last row that any lane wants) of a [*, row] matrix, D / 64 panels
template <int NP>
__device__ __forceinline__ void ap_tile_issue(const TileDma& d, const bf16* base, long long row, int r0, int last, bf16* tile, int wave) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const bf16* src = base + static_cast<long long>(min(r0 + static_cast<int>(d.row[j]), last)) * row + d.off[j];
#pragma unroll
        for (int pn = 0; pn < NP; ++pn)
            __builtin_amdgcn_global_load_lds((at_global_cvoid*)(src + 64 * pn), (at_lds_void*)(tile + pn * AT_TILE + (2 * wave + j) * 512), 16, 0, 0);
    }
}

// the values of reads issued by inline assembly, taken over behind the wait: nothing that uses them can move in front of it
__device__ __forceinline__ void taken(RowFrags& f) { asm volatile("" : "+v"(f.v[0]), "+v"(f.v[1]), "+v"(f.v[2]), "+v"(f.v[3])); }
__device__ __forceinline__ void taken(TrFrags& f) { asm volatile("" : "+v"(f.lo[0]), "+v"(f.lo[1]), "+v"(f.hi[0]), "+v"(f.hi[1])); }
__device__ __forceinline__ void taken(f32x4 (&f)[4]) { asm volatile("" : "+v"(f[0]), "+v"(f[1]), "+v"(f[2]), "+v"(f[3])); }

// ---- one row by a whole wave (lane = element lane, lane + 64), over its own interval only
template <int NP>
__device__ __forceinline__ void row_forward(const PackedArgs& p, int h, int row, int lane) {
    const int hk = h / p.group;
    const int2 s = ap_keys_of(p, row);
    float qv[NP], o[NP], m = -AP_INF, l = 0.f;
#pragma unroll
    for (int e = 0; e < NP; ++e) {
        qv[e] = bf16_to_f32(p.q[row * p.q_row + h * p.q_head + lane + 64 * e]);
        o[e] = 0.f;
    }
    for (int j = s.x; j < s.y; ++j) {
        float a = 0.f;
#pragma unroll
        for (int e = 0; e < NP; ++e) a += qv[e] * bf16_to_f32(p.k[j * p.k_row + hk * p.k_head + lane + 64 * e]);
        a = wave_sum(a) * p.scale_log2;
        const float mn = fmaxf(m, a), ref = mn == -AP_INF ? 0.f : mn;
        const float alpha = fast_exp2(m - ref), w = fast_exp2(a - ref);
        l = l * alpha + w;
#pragma unroll
        for (int e = 0; e < NP; ++e) o[e] = o[e] * alpha + w * bf16_to_f32(p.v[j * p.v_row + hk * p.v_head + lane + 64 * e]);
        m = mn;
    }
#pragma unroll
    for (int e = 0; e < NP; ++e) p.out[row * p.o_row + h * (64 * NP) + lane + 64 * e] = f32_to_bf16(o[e] / l);
    if (lane == 0) p.lse[static_cast<size_t>(h) * p.T + row] = log2f(l) + m;
}

template <int NP>
__device__ __forceinline__ void row_dq(const PackedArgs& p, int h, int row, int lane) {
    const int hk = h / p.group;
    const int2 s = ap_keys_of(p, row);
    const float lse = p.lse[static_cast<size_t>(h) * p.T + row];
    float qv[NP], dov[NP], dq[NP], dl = 0.f;
#pragma unroll
    for (int e = 0; e < NP; ++e) {
        const long long at = row * p.o_row + h * (64 * NP) + lane + 64 * e;
        qv[e] = bf16_to_f32(p.q[row * p.q_row + h * p.q_head + lane + 64 * e]);
        dov[e] = bf16_to_f32(p.dout[at]);
        dl += dov[e] * bf16_to_f32(p.o[at]);
        dq[e] = 0.f;
    }
    dl = wave_sum(dl);
    for (int j = s.x; j < s.y; ++j) {
        float a = 0.f, b = 0.f, kv[NP];
#pragma unroll
        for (int e = 0; e < NP; ++e) {
            kv[e] = bf16_to_f32(p.k[j * p.k_row + hk * p.k_head + lane + 64 * e]);
            a += qv[e] * kv[e];
            b += dov[e] * bf16_to_f32(p.v[j * p.v_row + hk * p.v_head + lane + 64 * e]);
        }
        a = wave_sum(a);
        b = wave_sum(b);
        const float ds = fast_exp2(a * p.scale_log2 - lse) * (b - dl);
#pragma unroll
        for (int e = 0; e < NP; ++e) dq[e] += ds * kv[e];
    }
#pragma unroll
    for (int e = 0; e < NP; ++e) p.dq[row * p.dq_row + h * p.dq_head + lane + 64 * e] = f32_to_bf16(dq[e] * p.scale);
}

// heads [h0, h1) of the key's group
template <int NP>
__device__ __forceinline__ void row_dkv(const PackedArgs& p, int hk, int h0, int h1, int split, int row, int lane) {
    const int2 s = ap_queries_of(p, row);
    float kv[NP], vv[NP], dk[NP], dv[NP];
#pragma unroll
    for (int e = 0; e < NP; ++e) {
        kv[e] = bf16_to_f32(p.k[row * p.k_row + hk * p.k_head + lane + 64 * e]);
        vv[e] = bf16_to_f32(p.v[row * p.v_row + hk * p.v_head + lane + 64 * e]);
        dk[e] = dv[e] = 0.f;
    }
    for (int h = h0; h < h1; ++h)
        for (int i = s.x; i < s.y; ++i) {
            float a = 0.f, b = 0.f, qv[NP], dov[NP];
#pragma unroll
            for (int e = 0; e < NP; ++e) {
                qv[e] = bf16_to_f32(p.q[i * p.q_row + h * p.q_head + lane + 64 * e]);
                dov[e] = bf16_to_f32(p.dout[i * p.o_row + h * (64 * NP) + lane + 64 * e]);
                a += qv[e] * kv[e];
                b += dov[e] * vv[e];
            }
            a = wave_sum(a);
            b = wave_sum(b);
            const float pr = fast_exp2(a * p.scale_log2 - p.lse[static_cast<size_t>(h) * p.T + i]);
            const float ds = pr * (b + p.delta[static_cast<size_t>(h) * p.T + i]);
#pragma unroll
            for (int e = 0; e < NP; ++e) {
                dk[e] += ds * qv[e];
                dv[e] += pr * dov[e];
            }
        }
#pragma unroll
    for (int e = 0; e < NP; ++e) {
        if (p.part != nullptr) {
            const size_t one = static_cast<size_t>(p.T) * p.Hk * (64 * NP);
            float* dst = p.part + static_cast<size_t>(split) * 2 * one + (static_cast<size_t>(row) * p.Hk + hk) * (64 * NP) + lane + 64 * e;
            dst[0] = dk[e] * p.scale;
            dst[one] = dv[e];
        } else {
            p.dk[row * p.dk_row + hk * p.dk_head + lane + 64 * e] = f32_to_bf16(dk[e] * p.scale);
            p.dv[row * p.dv_row + hk * p.dv_head + lane + 64 * e] = f32_to_bf16(dv[e]);
        }
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
// sizes.  Under a causal mask the blocks of a long sequence with the most tiles come first.
__device__ __forceinline__ void ap_unit(const PackedArgs& p, int heads, int& blk, int& h) {
    blk = blockIdx.x / heads;
    h = blockIdx.x - blk * heads;
    if (p.causal) blk = p.nblk - 1 - blk;
}

template <int NP>
__global__ __launch_bounds__(256, NP == 1 ? 3 : 2) void packed_fwd_kernel(const PackedArgs p) {
    constexpr int TILE = NP * AT_TILE, RING = ap_ring<NP>;
    extern __shared__ __attribute__((aligned(1024))) bf16 ap_smem[];
    bf16* sK = ap_smem;                    // [RING][TILE]
    bf16* sV = ap_smem + RING * TILE;   // [RING][TILE]
    __shared__ int sB[8];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int hi = lane >> 5, lq = lane & 31;
    int blk, h;
    ap_unit(p, p.H, blk, h);
    const int hk = h / p.group;
    const int qw0 = blk * AT_BR + 32 * wave, qrow = qw0 + lq;
    const int2 span = ap_keys_of(p, qrow);
    const Bounds wb = wave_bounds(span);
    if (lane == 0) {
        sB[wave] = wb.lo;
        sB[4 + wave] = wb.hi;
    }
    __syncthreads();
    const int k_lo = min(min(sB[0], sB[1]), min(sB[2], sB[3])), k_hi = max(max(sB[4], sB[5]), max(sB[6], sB[7]));
    const int nt = k_hi > k_lo ? (k_hi - k_lo + AT_T - 1) / AT_T : 0;
    const int t_lo = wb.hi > wb.lo ? (wb.lo - k_lo) / AT_T : nt, t_hi = wb.hi > wb.lo ? (wb.hi - k_lo + AT_T - 1) / AT_T : nt;
    const bf16* kbase = p.k + hk * p.k_head;
    const bf16* vbase = p.v + hk * p.v_head;
    const TileDma dma = tile_dma_setup(wave, lane);
    const FragAddr fa = frag_addr_setup(lane);

    bf16x8 qf[4 * NP];  // B operand of S^T
    {
        const bf16* qp = p.q + min(qrow, p.T - 1) * p.q_row + h * p.q_head + 8 * hi;
#pragma unroll
        for (int ks = 0; ks < 4 * NP; ++ks) qf[ks] = *reinterpret_cast<const bf16x8*>(qp + 16 * ks);
    }
    auto issue = [&](int t, int slot) {
        ap_tile_issue<NP>(dma, kbase, p.k_row, k_lo + t * AT_T, k_hi - 1, sK + slot * TILE, wave);
        ap_tile_issue<NP>(dma, vbase, p.v_row, k_lo + t * AT_T, k_hi - 1, sV + slot * TILE, wave);
    };
#pragma unroll
    for (int t = 0; t < RING - 1; ++t)
        if (t < nt) issue(t, t);

    f32x16 o[2 * NP];
#pragma unroll
    for (int d = 0; d < 2 * NP; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[d][e] = 0.f;
    float lsum = 0.f;      // this lane's share of the row sum
    float m = -AP_INF;     // running maximum (log2 units) ...
    float ref = 0.f;       // ... and what the exponents are taken about: the maximum, 0 before the first key
    const uint32_t sk_lds = lds_addr(sK), sv_lds = lds_addr(sV);

    int buf = 0;
    auto next_tile = [&](int t) {  // (the protocol of the fixed-length kernels)
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
        const uint32_t sk_tile = sk_lds + static_cast<uint32_t>(cur) * (TILE * 2), sv_tile = sv_lds + static_cast<uint32_t>(cur) * (TILE * 2);
        const bool masked = k0 < wb.max_lo || k0 + AT_T > wb.min_hi;
        const int rel_lo = span.x - k0 - 4 * hi;
        const uint32_t rel_n = static_cast<uint32_t>(span.y - span.x);  // offset o is valid: (unsigned)(o - rel_lo) < rel_n
        auto scores = [&](f32x16& acc, RowFrags(&kf)[NP]) {
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[e] = 0.f;
#pragma unroll
            for (int pn = 0; pn < NP; ++pn)
#pragma unroll
                for (int ks = 0; ks < 4; ++ks) acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(frag_rows_get(kf[pn], ks), qf[4 * pn + ks], acc, 0, 0, 0);
        };
        auto read_k = [&](RowFrags(&kf)[NP], const int kt) {
#pragma unroll
            for (int pn = 0; pn < NP; ++pn) frag_rows_issue(kf[pn], sk_tile + pn * (AT_TILE * 2), fa, kt);
        };
        auto take_k = [&](RowFrags(&kf)[NP]) {
#pragma unroll
            for (int pn = 0; pn < NP; ++pn) taken(kf[pn]);
        };
        auto read_v = [&](TrFrags(&vf)[2 * NP], const int kt) {
#pragma unroll
            for (int d = 0; d < 2 * NP; ++d) frag_tr_issue(vf[d], sv_tile + (d >> 1) * (AT_TILE * 2), fa, d & 1, kt);
        };
        auto take_v = [&](TrFrags(&vf)[2 * NP]) {
#pragma unroll
            for (int d = 0; d < 2 * NP; ++d) taken(vf[d]);
        };
        // scores -> probabilities about the running reference, in place; returns the lane's partial row sum.  Every lane's
        // first key lies in a half that starts at or before the wave's largest first key: those halves take the maximum;
        // later ones only when a partial sum outgrows 2^30 (the maximum rose by 30 octaves).
        auto probs = [&](f32x16& acc, const int koff, const bool careful) {
            if (masked) {
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    acc[r] = static_cast<uint32_t>(koff + (r & 3) + 8 * (r >> 2) - rel_lo) < rel_n ? acc[r] : -AP_INF;
            }
            if (careful) {
                float mx = acc[0];
#pragma unroll
                for (int r = 1; r < 16; ++r) mx = fmaxf(mx, acc[r]);
                mx = other_half_max(mx) * p.scale_log2;
                const float m_new = fmaxf(m, mx), next = m_new == -AP_INF ? 0.f : m_new;
                const float alpha = m == -AP_INF ? 0.f : fast_exp2(ref - next);  // (before the row's first key there is nothing to keep)
                lsum *= alpha;
#pragma unroll
                for (int d = 0; d < 2 * NP; ++d)
#pragma unroll
                    for (int e = 0; e < 16; ++e) o[d][e] *= alpha;
                m = m_new;
                ref = next;
            }
            float sum = 0.f;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                acc[r] = fast_exp2(fmaf(acc[r], p.scale_log2, -ref));
                sum += acc[r];
            }
            return sum;
        };
        auto softmax_half = [&](f32x16& acc, const int kt) {
            const bool careful = k0 + 32 * kt <= wb.max_lo;
            float ls = probs(acc, 32 * kt, careful);
            if (!careful && __builtin_expect(__any(!(ls <= 1073741824.f)), 0)) {
                RowFrags kf[NP];
                read_k(kf, kt);
                lds_wait<0>();
                take_k(kf);
                scores(acc, kf);
                ls = probs(acc, 32 * kt, true);
            }
            lsum += ls;
        };
        auto values = [&](const f32x16& acc, const TrFrags(&vf)[2 * NP]) {
            const bf16x8 pb0 = pack_half(acc, 0), pb1 = pack_half(acc, 1);
#pragma unroll
            for (int d = 0; d < 2 * NP; ++d) o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(frag_tr_get(vf[d], 0), pb0, o[d], 0, 0, 0);
#pragma unroll
            for (int d = 0; d < 2 * NP; ++d) o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(frag_tr_get(vf[d], 1), pb1, o[d], 0, 0, 0);
        };
        // two halves of 32 keys, so that the matrix pipe has work while the vector ALU turns scores into probabilities:
        //   S(0) S(1) | softmax(0) | PV(0) | softmax(1) | PV(1)
        f32x16 acc0, acc1;
        {
            RowFrags kf[NP];
            read_k(kf, 0);
            lds_wait<0>();
            take_k(kf);
            scores(acc0, kf);
            read_k(kf, 1);
            lds_wait<0>();
            take_k(kf);
            scores(acc1, kf);
        }
        TrFrags vf[2 * NP];
        read_v(vf, 0);
        softmax_half(acc0, 0);
        lds_wait<0>();
        take_v(vf);
        values(acc0, vf);
        read_v(vf, 1);
        softmax_half(acc1, 1);
        lds_wait<0>();
        take_v(vf);
        values(acc1, vf);
        __builtin_amdgcn_sched_barrier(0);
    }
    for (int t = max(t_lo, t_hi); t < nt; ++t) next_tile(t);
    asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
    const bool some = span.y > span.x;
    const float lt = other_half_sum(lsum);
    const float inv = some ? 1.f / lt : 0.f;
    if (!some) {
#pragma unroll
        for (int d = 0; d < 2 * NP; ++d)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[d][e] = 0.f;
    }
    if (hi == 0 && qrow < p.T) p.lse[static_cast<size_t>(h) * p.T + qrow] = some ? log2f(lt) + ref : 0.f;
    bf16* orow0 = p.out + qw0 * p.o_row + h * (64 * NP);
    bf16* so = sK + wave * (32 * AT_D);
#pragma unroll
    for (int pn = 0; pn < NP; ++pn)
        store_rows32(so, o + 2 * pn, inv, lane, p.T - qw0, [&](int row) { return orow0 + row * p.o_row + 64 * pn; });
    uint32_t bad = bad_rows(o, some);
    const unsigned long long bl = __ballot(some && !ap_finite(lt));
    bad |= static_cast<uint32_t>(bl) | static_cast<uint32_t>(bl >> 32);
    if (__builtin_expect(bad != 0, 0)) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the rows just stored are written over
        for (int r = 0; r < 32; ++r)
            if ((bad >> r) & 1) row_forward<NP>(p, h, qw0 + r, lane);
    }
}

template <int NP>
__global__ __launch_bounds__(256, NP == 1 ? 3 : 2) void packed_dq_kernel(const PackedArgs p) {
    constexpr int TILE = NP * AT_TILE, RING = ap_ring<NP>;
    extern __shared__ __attribute__((aligned(1024))) bf16 ap_smem[];
    bf16* sK = ap_smem;
    bf16* sV = ap_smem + RING * TILE;
    __shared__ int sB[8];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int hi = lane >> 5, lq = lane & 31;
    int blk, h;
    ap_unit(p, p.H, blk, h);
    const int hk = h / p.group;
    const int qw0 = blk * AT_BR + 32 * wave, qrow = qw0 + lq;
    const int2 span = ap_keys_of(p, qrow);
    const Bounds wb = wave_bounds(span);
    if (lane == 0) {
        sB[wave] = wb.lo;
        sB[4 + wave] = wb.hi;
    }
    __syncthreads();
    const int k_lo = min(min(sB[0], sB[1]), min(sB[2], sB[3])), k_hi = max(max(sB[4], sB[5]), max(sB[6], sB[7]));
    const int nt = k_hi > k_lo ? (k_hi - k_lo + AT_T - 1) / AT_T : 0;
    const int t_lo = wb.hi > wb.lo ? (wb.lo - k_lo) / AT_T : nt, t_hi = wb.hi > wb.lo ? (wb.hi - k_lo + AT_T - 1) / AT_T : nt;
    const bf16* kbase = p.k + hk * p.k_head;
    const bf16* vbase = p.v + hk * p.v_head;
    const TileDma dma = tile_dma_setup(wave, lane);
    const FragAddr fa = frag_addr_setup(lane);
    auto issue = [&](int t, int slot) {
        ap_tile_issue<NP>(dma, kbase, p.k_row, k_lo + t * AT_T, k_hi - 1, sK + slot * TILE, wave);
        ap_tile_issue<NP>(dma, vbase, p.v_row, k_lo + t * AT_T, k_hi - 1, sV + slot * TILE, wave);
    };
#pragma unroll
    for (int t = 0; t < RING - 1; ++t)
        if (t < nt) issue(t, t);
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
            const bf16x8 ov = *reinterpret_cast<const bf16x8*>(p.o + orow + 16 * ks);
#pragma unroll
            for (int e = 0; e < 8; ++e) dl += bf16_to_f32(dof[ks][e]) * bf16_to_f32(ov[e]);
        }
        ndl = -other_half_sum(dl);
        const size_t off = static_cast<size_t>(h) * p.T + qc;
        if (hi == 0 && qrow < p.T) p.delta[off] = ndl;
        nl = -p.lse[off];
    }
    f32x16 dq[2 * NP];
#pragma unroll
    for (int d = 0; d < 2 * NP; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) dq[d][e] = 0.f;
    const uint32_t sk_lds = lds_addr(sK), sv_lds = lds_addr(sV);

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
        const uint32_t sk_tile = sk_lds + static_cast<uint32_t>(cur) * (TILE * 2), sv_tile = sv_lds + static_cast<uint32_t>(cur) * (TILE * 2);
        const bool masked = k0 < wb.max_lo || k0 + AT_T > wb.min_hi;
        const int rel_lo = span.x - k0 - 4 * hi;
        const uint32_t rel_n = static_cast<uint32_t>(span.y - span.x);
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
            if (k0 + 32 * kt >= wb.hi || k0 + 32 * kt + 32 <= wb.lo) continue;  // a half that no row of the wave reaches
            f32x16 s, dp;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                s[e] = 0.f;
                dp[e] = ndl;
            }
            {
                RowFrags f[NP];
                auto read = [&](uint32_t tile) {
#pragma unroll
                    for (int pn = 0; pn < NP; ++pn) frag_rows_issue(f[pn], tile + pn * (AT_TILE * 2), fa, kt);
                    lds_wait<0>();
#pragma unroll
                    for (int pn = 0; pn < NP; ++pn) taken(f[pn]);
                };
                read(sk_tile);
#pragma unroll
                for (int ks = 0; ks < 4 * NP; ++ks) s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(frag_rows_get(f[ks >> 2], ks & 3), qf[ks], s, 0, 0, 0);
                read(sv_tile);  // (under the products just issued)
#pragma unroll
                for (int ks = 0; ks < 4 * NP; ++ks) dp = __builtin_amdgcn_mfma_f32_32x32x16_bf16(frag_rows_get(f[ks >> 2], ks & 3), dof[ks], dp, 0, 0, 0);
            }
            TrFrags kf[2 * NP];  // on their way during the vector work
#pragma unroll
            for (int d = 0; d < 2 * NP; ++d) frag_tr_issue(kf[d], sk_tile + (d >> 1) * (AT_TILE * 2), fa, d & 1, kt);
            if (masked) {
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    s[r] = static_cast<uint32_t>(32 * kt + (r & 3) + 8 * (r >> 2) - rel_lo) < rel_n ? s[r] : -AP_INF;
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = fast_exp2(fmaf(s[r], p.scale_log2, nl)) * dp[r];
            const bf16x8 ds0 = pack_half(s, 0), ds1 = pack_half(s, 1);
            lds_wait<0>();
#pragma unroll
            for (int d = 0; d < 2 * NP; ++d) {
                taken(kf[d]);
                dq[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(frag_tr_get(kf[d], 0), ds0, dq[d], 0, 0, 0);
                dq[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(frag_tr_get(kf[d], 1), ds1, dq[d], 0, 0, 0);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
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
    bf16* drow0 = p.dq + qw0 * p.dq_row + h * p.dq_head;
    bf16* so = sK + wave * (32 * AT_D);
#pragma unroll
    for (int pn = 0; pn < NP; ++pn)
        store_rows32(so, dq + 2 * pn, p.scale, lane, p.T - qw0, [&](int row) { return drow0 + row * p.dq_row + 64 * pn; });
    const uint32_t bad = bad_rows(dq, some);
    if (__builtin_expect(bad != 0, 0)) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        for (int r = 0; r < 32; ++r)
            if ((bad >> r) & 1) row_dq<NP>(p, h, qw0 + r, lane);
    }
}

template <int NP>
__global__ __launch_bounds__(256, NP == 1 ? 2 : 1) void packed_dkv_kernel(const PackedArgs p) {
    constexpr int TILE = NP * AT_TILE;
    extern __shared__ __attribute__((aligned(1024))) bf16 ap_smem[];
    bf16* sQ = ap_smem;
    bf16* sDO = ap_smem + AT_RING * TILE;
    __shared__ __attribute__((aligned(1024))) float sRow[AT_RING][4][AT_T];  // per tile: lse, -delta, two unused rows (waves 2, 3)
    __shared__ int sB[8];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int hi = lane >> 5, lq = lane & 31;
    int blk, u;
    ap_unit(p, p.Hk * p.splits, blk, u);
    if (p.causal) blk = p.nblk - 1 - blk;  // here the first key blocks carry the most query tiles
    const int hk = u / p.splits, split = u - hk * p.splits;
    const int h0 = hk * p.group + split * p.group / p.splits, h1 = hk * p.group + (split + 1) * p.group / p.splits;
    const int kw0 = blk * AT_BR + 32 * wave, key = kw0 + lq;
    const int2 span = ap_queries_of(p, key);
    const Bounds wb = wave_bounds(span);
    if (lane == 0) {
        sB[wave] = wb.lo;
        sB[4 + wave] = wb.hi;
    }
    __syncthreads();
    const int q_lo = min(min(sB[0], sB[1]), min(sB[2], sB[3])), q_hi = max(max(sB[4], sB[5]), max(sB[6], sB[7]));
    const int nt1 = q_hi > q_lo ? (q_hi - q_lo + AT_T - 1) / AT_T : 0;  // tiles of one head; the heads follow each other
    const int nt = nt1 * (h1 - h0);
    const int t_lo = wb.hi > wb.lo ? (wb.lo - q_lo) / AT_T : nt1, t_hi = wb.hi > wb.lo ? (wb.hi - q_lo + AT_T - 1) / AT_T : nt1;
    const TileDma dma = tile_dma_setup(wave, lane);
    const FragAddr fa = frag_addr_setup(lane);
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
        ap_tile_issue<NP>(dma, p.q + is_h * p.q_head, p.q_row, r0, q_hi - 1, sQ + slot * TILE, wave);
        ap_tile_issue<NP>(dma, p.dout + is_h * (64 * NP), p.o_row, r0, q_hi - 1, sDO + slot * TILE, wave);
        const float* rows = (wave & 1 ? p.delta : p.lse) + static_cast<size_t>(is_h) * p.T;
        __builtin_amdgcn_global_load_lds((at_global_cvoid*)(rows + min(r0 + lane, q_hi - 1)), (at_lds_void*)&sRow[slot][wave][0], 4, 0, 0);
        if (++is_t == nt1) {
            is_t = 0;
            ++is_h;
        }
    };
#pragma unroll
    for (int i = 0; i < 2; ++i)
        if (i < nt) issue(i);
    f32x16 dk[2 * NP], dv[2 * NP];
#pragma unroll
    for (int d = 0; d < 2 * NP; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) dk[d][e] = dv[d][e] = 0.f;
    const uint32_t sq_lds = lds_addr(sQ), sdo_lds = lds_addr(sDO), srow_lds = lds_addr(&sRow[0][0][0]);

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
            const uint32_t sq_tile = sq_lds + static_cast<uint32_t>(cur) * (TILE * 2), sdo_tile = sdo_lds + static_cast<uint32_t>(cur) * (TILE * 2);
            const uint32_t row_tile = srow_lds + static_cast<uint32_t>(cur) * (4 * AT_T * 4) + 16 * hi;
            const bool masked = q0 < wb.max_lo || q0 + AT_T > wb.min_hi;
            const int rel_lo = span.x - q0 - 4 * hi;
            const uint32_t rel_n = static_cast<uint32_t>(span.y - span.x);
            // S and dP of a half of 32 queries
            auto products = [&](f32x16& s, f32x16& dp, const int qt) {
                f32x4 nd[4];
                RowFrags qf[NP], dof[NP];
#pragma unroll
                for (int r4 = 0; r4 < 4; ++r4) lds_read_f32x4(nd[r4], row_tile + AT_T * 4 + (32 * qt + 8 * r4) * 4);
#pragma unroll
                for (int pn = 0; pn < NP; ++pn) frag_rows_issue(qf[pn], sq_tile + pn * (AT_TILE * 2), fa, qt);
#pragma unroll
                for (int pn = 0; pn < NP; ++pn) frag_rows_issue(dof[pn], sdo_tile + pn * (AT_TILE * 2), fa, qt);
                lds_wait<4 * NP>();
                taken(nd);
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    s[e] = 0.f;
                    dp[e] = nd[e >> 2][e & 3];
                }
#pragma unroll
                for (int pn = 0; pn < NP; ++pn) {
                    taken(qf[pn]);
#pragma unroll
                    for (int ks = 0; ks < 4; ++ks) s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(frag_rows_get(qf[pn], ks), kf[4 * pn + ks], s, 0, 0, 0);
                }
                lds_wait<0>();
#pragma unroll
                for (int pn = 0; pn < NP; ++pn) {
                    taken(dof[pn]);
#pragma unroll
                    for (int ks = 0; ks < 4; ++ks) dp = __builtin_amdgcn_mfma_f32_32x32x16_bf16(frag_rows_get(dof[pn], ks), vf[4 * pn + ks], dp, 0, 0, 0);
                }
            };
            auto finish = [&](f32x16& s, f32x16& dp, const int qt) {
                f32x4 l2[4];
#pragma unroll
                for (int r4 = 0; r4 < 4; ++r4) lds_read_f32x4(l2[r4], row_tile + (32 * qt + 8 * r4) * 4);
                TrFrags dot[2], qtf[2];  // two column tiles of dO^T and Q^T at a time, on their way during the vector work
#pragma unroll
                for (int d = 0; d < 2; ++d) {
                    frag_tr_issue(dot[d], sdo_tile, fa, d, qt);
                    frag_tr_issue(qtf[d], sq_tile, fa, d, qt);
                }
                lds_wait<15>();  // (the row terms are the oldest four of twenty reads; the counter ends at 15)
                taken(l2);
                if (masked) {
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        s[r] = static_cast<uint32_t>(32 * qt + (r & 3) + 8 * (r >> 2) - rel_lo) < rel_n ? s[r] : -AP_INF;
                }
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    s[r] = fast_exp2(fmaf(s[r], p.scale_log2, -l2[r >> 2][r & 3]));
                    dp[r] *= s[r];
                }
                bf16x8 pb[2], dsb[2];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    pb[j] = pack_half(s, j);
                    dsb[j] = pack_half(dp, j);
                }
#pragma unroll
                for (int pn = 0; pn < NP; ++pn) {
                    lds_wait<0>();
                    bf16x8 da[2][2], qa[2][2];
#pragma unroll
                    for (int d = 0; d < 2; ++d) {
                        taken(dot[d]);
                        taken(qtf[d]);
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            da[d][j] = frag_tr_get(dot[d], j);
                            qa[d][j] = frag_tr_get(qtf[d], j);
                        }
                    }
                    if (pn + 1 < NP) {
#pragma unroll
                        for (int d = 0; d < 2; ++d) {
                            frag_tr_issue(dot[d], sdo_tile + (pn + 1) * (AT_TILE * 2), fa, d, qt);
                            frag_tr_issue(qtf[d], sq_tile + (pn + 1) * (AT_TILE * 2), fa, d, qt);
                        }
                    }
#pragma unroll
                    for (int d = 0; d < 2; ++d)
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            dv[2 * pn + d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(da[d][j], pb[j], dv[2 * pn + d], 0, 0, 0);
                            dk[2 * pn + d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(qa[d][j], dsb[j], dk[2 * pn + d], 0, 0, 0);
                        }
                }
            };
            // (halves that no key of the wave meets are left out)
            f32x16 s, dp;
            if (q0 + 32 > wb.lo) {
                products(s, dp, 0);
                finish(s, dp, 0);
            }
            if (q0 + 32 < wb.hi) {
                products(s, dp, 1);
                finish(s, dp, 1);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
    const bool some = span.y > span.x;
    if (!some) {
#pragma unroll
        for (int d = 0; d < 2 * NP; ++d)
#pragma unroll
            for (int e = 0; e < 16; ++e) dk[d][e] = dv[d][e] = 0.f;
    }
    if (p.part != nullptr) {
        const size_t one = static_cast<size_t>(p.T) * p.Hk * (64 * NP);
        float* dst = p.part + static_cast<size_t>(split) * 2 * one + (static_cast<size_t>(key) * p.Hk + hk) * (64 * NP) + 4 * hi;
        if (key < p.T) {
#pragma unroll
            for (int d = 0; d < 2 * NP; ++d)
#pragma unroll
                for (int r4 = 0; r4 < 4; ++r4) {
                    f32x4 a, b;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        a[e] = dk[d][4 * r4 + e] * p.scale;
                        b[e] = dv[d][4 * r4 + e];
                    }
                    *reinterpret_cast<f32x4*>(dst + 32 * d + 8 * r4) = a;
                    *reinterpret_cast<f32x4*>(dst + one + 32 * d + 8 * r4) = b;
                }
        }
    } else {
        bf16* so = sQ + wave * (32 * AT_D);
        bf16* krow0 = p.dk + kw0 * p.dk_row + hk * p.dk_head;
        bf16* vrow0 = p.dv + kw0 * p.dv_row + hk * p.dv_head;
#pragma unroll
        for (int pn = 0; pn < NP; ++pn) {
            store_rows32(so, dk + 2 * pn, p.scale, lane, p.T - kw0, [&](int row) { return krow0 + row * p.dk_row + 64 * pn; });
            store_rows32(so, dv + 2 * pn, 1.f, lane, p.T - kw0, [&](int row) { return vrow0 + row * p.dv_row + 64 * pn; });
        }
    }
    const uint32_t bad = bad_rows(dk, some) | bad_rows(dv, some);
    if (__builtin_expect(bad != 0, 0)) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        for (int r = 0; r < 32; ++r)
            if ((bad >> r) & 1) row_dkv<NP>(p, hk, h0, h1, split, kw0 + r, lane);
    }
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

// Sequence of every row: offsets[s] <= row < offsets[s + 1], cut to the rows there are.  The last sequence that starts at or
// before the row is the only one that can hold it (empty sequences share their start with the one behind them).
__global__ __launch_bounds__(256) void pack_spans_kernel(const int* __restrict__ offsets, int n, int rows, int2* __restrict__ spans,
                                                        long long* __restrict__ positions) {
    const int row = blockIdx.x * 256 + threadIdx.x;
    if (row >= rows) return;
    int lo = 0, hi = n;  // offsets[0 .. lo) start at or before the row
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (offsets[mid] <= row) lo = mid + 1;
        else hi = mid;
    }
    int2 s = {0, 0};
    if (lo > 0) {
        const int first = max(offsets[lo - 1], 0), end = min(offsets[lo], rows);
        if (row < end) s = {first, end};
    }
    spans[row] = s;
    positions[row] = s.y > 0 ? row - s.x : 0;
}

// offsets: [sequences + 1] int32, not falling.
PDT_API int pdt_pack_spans(const int* offsets, int sequences, int rows, void* spans, long long* positions, void* stream) {
    if (sequences < 0 || rows <= 0) return -1;
    hipLaunchKernelGGL(pack_spans_kernel, dim3(pdt_cdiv(rows, 256)), dim3(256), 0, static_cast<hipStream_t>(stream), offsets, sequences, rows,
                       static_cast<int2*>(spans), positions);
    return pdt_launch_status();
}

static bool ap_stride_ok(const long long* st, int n) {
    for (int i = 0; i < n; ++i)
        if (st[i] <= 0 || (st[i] % 8) != 0) return false;
    return true;
}

static int ap_args(PackedArgs& a, const void* spans, int T, int H, int Hk, int D, float scale, int causal) {
    if (T <= 0 || H <= 0 || Hk <= 0 || H % Hk != 0 || (D != 64 && D != 128) || !(scale > 0.f) || !(scale < 3.0e38f)) return -1;
    a.spans = static_cast<const int2*>(spans);
    a.T = T; a.H = H; a.Hk = Hk;
    a.group = H / Hk;
    a.nblk = pdt_cdiv(T, AT_BR);
    a.causal = causal != 0;
    a.splits = 1;
    a.scale = scale;
    a.scale_log2 = scale * 1.4426950408889634f;
    if (static_cast<long long>(a.nblk) * H >= (1ll << 31) || T >= (1 << 30)) return -1;
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
static int ap_launch(K kernel, unsigned long long& granted, unsigned grid, size_t lds, hipStream_t stream, const PackedArgs& a) {
    if (int e = ap_lds(kernel, lds, granted)) return e;
    hipLaunchKernelGGL(kernel, dim3(grid), dim3(256), lds, stream, a);
    return pdt_launch_status();
}

// st: row and head strides of q, k, v in elements (multiples of 8; 16-byte aligned pointers); out is [T, H, D] without gaps.
PDT_API int pdt_packed_attention_fwd(const void* q, const void* k, const void* v, void* out, float* lse, const void* spans, const long long* st,
                                     int T, int H, int Hk, int D, float scale, int causal, void* stream) {
    PackedArgs a = {};
    if (ap_args(a, spans, T, H, Hk, D, scale, causal) != 0 || !ap_stride_ok(st, 6)) return -1;
    a.q = static_cast<const bf16*>(q);
    a.k = static_cast<const bf16*>(k);
    a.v = static_cast<const bf16*>(v);
    a.out = static_cast<bf16*>(out);
    a.lse = lse;
    a.q_row = st[0]; a.q_head = st[1];
    a.k_row = st[2]; a.k_head = st[3];
    a.v_row = st[4]; a.v_head = st[5];
    a.o_row = static_cast<long long>(H) * D;
    const size_t lds = static_cast<size_t>(2 * (D == 64 ? ap_ring<1> : ap_ring<2>)) * AT_T * D * sizeof(bf16);
    const unsigned grid = static_cast<unsigned>(a.nblk) * H;
    static unsigned long long granted[2];
    return D == 64 ? ap_launch(packed_fwd_kernel<1>, granted[0], grid, lds, static_cast<hipStream_t>(stream), a)
                   : ap_launch(packed_fwd_kernel<2>, granted[1], grid, lds, static_cast<hipStream_t>(stream), a);
}

// How many ways the backward pass splits the query heads of a key head (1: no partial sums).  A key block with all the
// heads of its group is one workgroup; with few key heads that leaves CUs idle.
PDT_API int pdt_packed_attention_splits(int T, int H, int Hk) {
    const int group = H / Hk, units = pdt_cdiv(T, AT_BR) * Hk;
    int s = 1;
    while (s < group && units * s < 512) s *= 2;
    return s < group ? s : group;
}

// st: row and head strides of q, k, v, dq, dk, dv; o and dout are [T, H, D] without gaps.  delta: scratch, H * T floats.
// part: scratch, splits * 2 * T * Hk * D floats, unused (may be nullptr) where splits is 1.
PDT_API int pdt_packed_attention_bwd(const void* q, const void* k, const void* v, const void* o, const void* dout, const float* lse, float* delta,
                                     void* dq, void* dk, void* dv, float* part, int splits, const void* spans, const long long* st, int T, int H,
                                     int Hk, int D, float scale, int causal, void* stream) {
    PackedArgs a = {};
    if (ap_args(a, spans, T, H, Hk, D, scale, causal) != 0 || !ap_stride_ok(st, 12)) return -1;
    if (splits < 1 || splits > a.group || (splits > 1 && part == nullptr) || static_cast<long long>(a.nblk) * Hk * splits >= (1ll << 31)) return -1;
    a.q = static_cast<const bf16*>(q);
    a.k = static_cast<const bf16*>(k);
    a.v = static_cast<const bf16*>(v);
    a.o = static_cast<const bf16*>(o);
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
    const size_t lds_k = static_cast<size_t>(2 * AT_RING) * AT_T * D * sizeof(bf16);
    const unsigned gq = static_cast<unsigned>(a.nblk) * H, gk = static_cast<unsigned>(a.nblk) * Hk * splits;
    static unsigned long long granted[4];
    int rc = D == 64 ? ap_launch(packed_dq_kernel<1>, granted[0], gq, lds, s, a) : ap_launch(packed_dq_kernel<2>, granted[1], gq, lds, s, a);
    if (rc == 0) rc = D == 64 ? ap_launch(packed_dkv_kernel<1>, granted[2], gk, lds_k, s, a) : ap_launch(packed_dkv_kernel<2>, granted[3], gk, lds_k, s, a);
    if (rc != 0) return rc;
    if (a.part != nullptr) {
        const long long n = 2ll * T * Hk * D / 4;
        hipLaunchKernelGGL(packed_join_kernel, dim3(static_cast<unsigned>(n / 256 + 1 < 4096 ? n / 256 + 1 : 4096)), dim3(256), 0, s, a, D);
    }
    return pdt_launch_status();
}
