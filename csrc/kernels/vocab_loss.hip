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
// are joined, one pass turns the exponentials into q - p in place, and two more products give dx = (q - p) W and
// dW = (q - p)^T x; the factor tau / rows is applied to their fp32 sums.
#include "common.h"

typedef __attribute__((address_space(3))) void vl_lds_void;
typedef const __attribute__((address_space(1))) void vl_global_cvoid;

#define VL_INF __builtin_inff()
#define VL_GROUP 64   // vocabulary entries that share a maximum
#define VL_MAX_TOP 1024

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
// ------------------------------------------------------------------------------------------------
struct VocabGemm {
    const bf16 *a, *b;
    long long lda, ldb;
    int M, N, K;
    int tiles_m, tiles_n;
    const bf16* zeros;     // 16 bytes of zeros
    // scores
    float2* stats;         // [M][groups] {maximum (log2 units), sum}
    bf16* e;               // [M][lde] exponentials, or nullptr
    long long lde;
    int groups;
    float scale_log2;      // log2(e) / tau
    // dx, dW
    const float* alpha;    // device factor of the result
    bf16* out;             // bf16 result, or nullptr
    float* out32;          // fp32 result; split products: [splits][M][N] partial sums
    long long ldo;
    int accumulate;        // add to out32
    int k_per_split;       // multiple of 64
};

template <bool KMAJOR>
__device__ __forceinline__ int vl_swz(int row) { return KMAJOR ? (row & 3) | ((row >> 1) & 4) : row & 7; }

template <int KIND>
__global__ __launch_bounds__(512) void vocab_gemm_kernel(const VocabGemm p) {
    constexpr bool A_KM = KIND == 2, B_KM = KIND != 0;
    constexpr int STAGE = 2 * 256 * 64;  // elements: [A tile | B tile]
    extern __shared__ __attribute__((aligned(1024))) bf16 vl_smem[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave >> 2, wn = wave & 3;
    const int r16 = lane & 15, g4 = lane >> 4;

    // tiles in groups of eight rows of tiles: the 32 tiles an XCD works on at a time share 8 A and 4 B panels
    const int total = p.tiles_m * p.tiles_n;
    const int lin = xcd_remap(blockIdx.x, gridDim.x), split = lin / total, u = lin - split * total;
    const int per = 8 * p.tiles_n, grp = u / per, gm = min(8, p.tiles_m - grp * 8), in = u - grp * per;
    const int m0 = (grp * 8 + in % gm) * 256, n0 = (in / gm) * 256;
    const int k_lo = split * p.k_per_split, k_hi = min(p.K, k_lo + p.k_per_split);
    const int nsteps = (k_hi - k_lo + 63) / 64;

    // this lane's source of DMA piece i (four pieces of 1 KB per wave, operand and K-step) at k = 0
    const bf16 *a_src[4], *b_src[4];
    int a_k[4], b_k[4];  // K-major: the piece's row (its k inside the step)
    auto setup = [&](const bf16* base, long long ld, int first, int count, bool km, const bf16*(&src)[4], int(&k)[4]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (km) {
                const int row = (wave * 4 + i) * 2 + (lane >> 5), pc = lane & 31;
                const int col = (((pc >> 1) ^ vl_swz<true>(row)) << 4) | ((pc & 1) << 3);
                const int last = (count - 1) & ~7;  // (rows have multiples of 8 elements: the last chunk is whole)
                src[i] = base + min(first + col, last);
                k[i] = row;
            } else {
                const int row = (wave * 4 + i) * 8 + (lane >> 3), slot = lane & 7;
                src[i] = base + static_cast<long long>(min(first + row, count - 1)) * ld + ((slot ^ vl_swz<false>(row)) << 3);
                k[i] = 0;
            }
        }
    };
    setup(p.a, p.lda, m0, p.M, A_KM, a_src, a_k);
    setup(p.b, p.ldb, n0, p.N, B_KM, b_src, b_k);
    auto issue = [&](int s) {
        const int k0 = k_lo + s * 64;
        bf16* sA = vl_smem + (s & 1) * STAGE;
        bf16* sB = sA + 256 * 64;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const bf16* src;
            // k beyond the end: zeros from A, so that whatever B holds there does not count (B repeats its last row)
            if (A_KM) src = k0 + a_k[i] < k_hi ? a_src[i] + static_cast<long long>(k0 + a_k[i]) * p.lda : p.zeros;
            else src = a_src[i] + k0;
            __builtin_amdgcn_global_load_lds((vl_global_cvoid*)src, (vl_lds_void*)(sA + (wave * 4 + i) * 512), 16, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const bf16* src = B_KM ? b_src[i] + static_cast<long long>(min(k0 + b_k[i], p.K - 1)) * p.ldb : b_src[i] + k0;
            __builtin_amdgcn_global_load_lds((vl_global_cvoid*)src, (vl_lds_void*)(sB + (wave * 4 + i) * 512), 16, 0, 0);
        }
    };
    auto fragment = [&](const bf16* tile, int first, int kk, bool km) -> bf16x8 {
        if (km) {
            const int row = kk * 32 + 8 * g4 + ((lane >> 2) & 3);  // (rows row and row + 4 are swizzled alike)
            const bf16* at = tile + row * 256 + (((first >> 4) ^ vl_swz<true>(row)) << 4) + 4 * (lane & 3);
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)at);
            const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(at + 4 * 256));
            const s16x8 v = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
            return __builtin_bit_cast(bf16x8, v);
        }
        const int row = first + r16;
        return *reinterpret_cast<const bf16x8*>(tile + row * 64 + (((kk * 4 + g4) ^ vl_swz<false>(row)) << 3));
    };

    f32x4 acc[8][4];
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (nsteps > 0) issue(0);
    for (int s = 0; s < nsteps; ++s) {
        asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
        if (s + 1 < nsteps) issue(s + 1);
        const bf16* sA = vl_smem + (s & 1) * STAGE;
        const bf16* sB = sA + 256 * 64;
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            bf16x8 fb[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) fb[j] = fragment(sB, wn * 64 + j * 16, kk, B_KM);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const bf16x8 fa = fragment(sA, wm * 128 + i * 16, kk, A_KM);
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fb[j], fa, acc[i][j], 0, 0, 0);
            }
        }
    }
    asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
    // lane: row m = 16 i + (lane & 15), columns n = 16 j + 4 (lane >> 4) + 0 .. 3 of the wave's 128 x 64
    bf16* stage = vl_smem + wave * (16 * 64);  // 16 rows of the wave at a time, as whole 128-byte rows
    const int mw = m0 + wm * 128, nw = n0 + wn * 64;
    float alpha = 1.f;
    if constexpr (KIND != 0) alpha = p.out32 != nullptr && gridDim.x > static_cast<unsigned>(total) ? 1.f : p.alpha[0];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int m = mw + i * 16 + r16;
        if constexpr (KIND == 0) {
            float mx = -VL_INF;
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    acc[i][j][e] = nw + j * 16 + 4 * g4 + e < p.N ? acc[i][j][e] * p.scale_log2 : -VL_INF;
                    mx = fmaxf(mx, acc[i][j][e]);
                }
            mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
            mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
            const float ref = mx == -VL_INF ? 0.f : mx;  // (a group beyond the vocabulary, or one that is masked out)
            float sum = 0.f;
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    acc[i][j][e] = vl_exp2(acc[i][j][e] - ref);
                    sum += acc[i][j][e];
                }
            sum += __shfl_xor(sum, 16, 64);
            sum += __shfl_xor(sum, 32, 64);
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
                    if (mm < p.M && nn < p.lde) *reinterpret_cast<bf16x8*>(p.e + mm * p.lde + nn) = v;
                } else {
                    if (mm < p.M && nn < p.N) *reinterpret_cast<bf16x8*>(p.out + mm * p.ldo + nn) = v;
                }
            }
        } else if (m < p.M) {
            float* dst = p.out32 + static_cast<size_t>(split) * p.M * p.ldo + m * p.ldo + nw + 4 * g4;
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

// out = alpha * (sum of the split product's parts, in order)
__global__ __launch_bounds__(256) void vocab_join_kernel(const float* __restrict__ part, int splits, long long n, const float* __restrict__ alpha,
                                                        bf16* __restrict__ out) {
    const float a = alpha[0];
    for (long long i = (blockIdx.x * 256ll + threadIdx.x) * 4; i < n; i += gridDim.x * 1024ll) {
        f32x4 s = {0.f, 0.f, 0.f, 0.f};
        for (int k = 0; k < splits; ++k) s += *reinterpret_cast<const f32x4*>(part + k * n + i);
        bf16x4 r;
#pragma unroll
        for (int e = 0; e < 4; ++e) r[e] = f32_to_bf16(s[e] * a);
        *reinterpret_cast<bf16x4*>(out + i) = r;
    }
}

// ------------------------------------------------------------------------------------------------
// targets: weights p, base = sum p ln p (- sum p z / tau behind a projection), whether the row has a target
// ------------------------------------------------------------------------------------------------
struct Targets {
    const long long* ids;    // [rows][top]
    const float* teacher;    // [rows][top], or nullptr: one target of weight 1 (labels)
    float* p;                // [rows][top], unused for labels
    float* base;             // [rows]
    int* valid;              // [rows]
    const bf16 *x, *w;       // behind a projection: [rows][width], [vocab][width]; else nullptr
    bf16* x_used;            // copy of x with zeros in the rows without a target, or nullptr: what such a row holds (NaN, say)
                             // must not meet its zero gradient in the product that gives dW
    int rows, top, width;
    long long vocab;
    float inv_tau;
};

__device__ __forceinline__ float vl_dot8(const bf16* a, const bf16* b, float s) {
    const bf16x8 u = *reinterpret_cast<const bf16x8*>(a), v = *reinterpret_cast<const bf16x8*>(b);
#pragma unroll
    for (int e = 0; e < 8; ++e) s = fmaf(bf16_to_f32(u[e]), bf16_to_f32(v[e]), s);
    return s;
}

// one wave per row
__global__ __launch_bounds__(256) void vocab_targets_kernel(const Targets t) {
    const int lane = threadIdx.x & 63, row = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= t.rows) return;
    const long long* ids = t.ids + static_cast<size_t>(row) * t.top;
    auto present = [&](int k) { return ids[k] >= 0 && ids[k] < t.vocab; };
    float base = 0.f;
    bool some = false;
    if (t.teacher == nullptr) {
        some = present(0);
    } else {
        const float* z = t.teacher + static_cast<size_t>(row) * t.top;
        float* p = t.p + static_cast<size_t>(row) * t.top;
        float mx = -VL_INF;
        bool any = false;
        for (int k = lane; k < t.top; k += 64)
            if (present(k)) {
                any |= !(z[k] == -VL_INF);  // (NaN counts: it is to be seen in the loss)
                mx = fmaxf(mx, z[k]);
            }
        mx = wave_max(mx);
        some = __any(any);
        if (mx == -VL_INF) mx = 0.f;
        float sum = 0.f;
        for (int k = lane; k < t.top; k += 64)
            if (present(k)) sum += vl_exp2((z[k] - mx) * t.inv_tau * VL_LOG2E);
        sum = wave_sum(sum);
        const float ls = log2f(sum), inv = some ? 1.f / sum : 0.f;
        for (int k = lane; k < t.top; k += 64) {
            const float l = (z[k] - mx) * t.inv_tau * VL_LOG2E, pk = present(k) && some ? vl_exp2(l) * inv : 0.f;
            p[k] = pk;
            if (pk != 0.f) base += pk * (l - ls) * VL_LN2;
        }
        __threadfence_block();  // (the weights are read again by all lanes below)
    }
    if (t.x != nullptr && some) {
        const bf16* x = t.x + static_cast<size_t>(row) * t.width;
        for (int k = 0; k < t.top; ++k) {
            const float pk = t.teacher == nullptr ? 1.f : t.p[static_cast<size_t>(row) * t.top + k];
            if (pk == 0.f || !present(k)) continue;
            const bf16* w = t.w + ids[k] * t.width;
            float s = 0.f;
            for (int c = lane * 8; c < t.width; c += 512) s = vl_dot8(x + c, w + c, s);
            base -= pk * s * t.inv_tau;
        }
    }
    if (t.x_used != nullptr)
        for (int c = lane * 8; c < t.width; c += 512) {
            const size_t at = static_cast<size_t>(row) * t.width + c;
            *reinterpret_cast<bf16x8*>(t.x_used + at) = some ? *reinterpret_cast<const bf16x8*>(t.x + at) : bf16x8{};
        }
    base = wave_sum(base);
    if (lane == 0) {
        t.base[row] = base;
        t.valid[row] = some ? 1 : 0;
    }
}

// scal[0] = tau / rows with a target (0 without any), scal[1] = tau^2 / rows with a target
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
        scal[1] = n > 0 ? tau * tau / n : 0.f;
    }
}

__global__ __launch_bounds__(1024) void vocab_mean_kernel(const float* __restrict__ row_loss, int rows, const float* __restrict__ scal,
                                                         float* __restrict__ loss) {
    __shared__ float red[16];
    float s = 0.f;
    for (int i = threadIdx.x; i < rows; i += 1024) s += row_loss[i];
    s = block_sum(s, red);
    if (threadIdx.x == 0) loss[0] = s * scal[1];
}

// Targets of a row into LDS: id, and the weight of the id (entries that repeat an id add to its first place; others 0).
// Returns through `own` whether this thread's entry k is the one that writes the id.
struct TargetLds {
    int id[VL_MAX_TOP];
    float p[VL_MAX_TOP];
};
__device__ __forceinline__ void vl_load_targets(TargetLds& s, const long long* ids, const float* p, int top, long long vocab) {
    for (int k = threadIdx.x; k < top; k += blockDim.x) {
        const bool ok = ids[k] >= 0 && ids[k] < vocab;
        s.id[k] = ok ? static_cast<int>(ids[k]) : -1;
        s.p[k] = p != nullptr ? p[k] : 1.f;
    }
    __syncthreads();
}
__device__ __forceinline__ bool vl_merged(const TargetLds& s, int k, int top, float& p) {
    const int id = s.id[k];
    if (id < 0) return false;
    p = 0.f;
    for (int j = 0; j < top; ++j)
        if (s.id[j] == id) {
            if (j < k) return false;
            p += s.p[j];
        }
    return true;
}

// ---- behind a projection: one workgroup per row joins the groups; training: exponentials -> q - p in place
struct Rows {
    const float2* stats;
    bf16* e;
    long long lde;
    const long long* ids;
    const float* p;          // nullptr: labels
    const float* base;
    const int* valid;
    float* row_loss;
    int groups, top;
    long long vocab;
};

__global__ __launch_bounds__(256) void vocab_rows_kernel(const Rows a) {
    __shared__ float red[16];
    __shared__ TargetLds tg;
    const int row = blockIdx.x, tid = threadIdx.x;
    const float2* st = a.stats + static_cast<size_t>(row) * a.groups;
    float m = -VL_INF;
    for (int g = tid; g < a.groups; g += 256) m = fmaxf(m, st[g].x);
    m = block_max(m, red);
    const float ref = m == -VL_INF ? 0.f : m;
    float s = 0.f;
    for (int g = tid; g < a.groups; g += 256) s += st[g].y * vl_exp2(st[g].x - ref);
    s = block_sum(s, red);
    const float lse = ref + log2f(s);
    const bool valid = a.valid[row] != 0;
    if (tid == 0) a.row_loss[row] = valid ? a.base[row] + lse * VL_LN2 : 0.f;
    if (a.e == nullptr) return;
    bf16* e = a.e + row * a.lde;
    if (!valid) {
        for (long long c = tid * 8; c < a.lde; c += 2048) *reinterpret_cast<bf16x8*>(e + c) = bf16x8{};
        return;
    }
    vl_load_targets(tg, a.ids + static_cast<size_t>(row) * a.top, a.p == nullptr ? nullptr : a.p + static_cast<size_t>(row) * a.top, a.top, a.vocab);
    float val[VL_MAX_TOP / 256];
    uint32_t mine = 0;
#pragma unroll
    for (int i = 0; i < VL_MAX_TOP / 256; ++i) {
        const int k = tid + i * 256;
        float p;
        if (k < a.top && vl_merged(tg, k, a.top, p)) {
            const int id = tg.id[k];
            val[i] = bf16_to_f32(e[id]) * vl_exp2(st[id >> 6].x - lse) - p;
            mine |= 1u << i;
        }
    }
    __syncthreads();  // the targets' exponentials are read
    for (long long c = tid * 8; c < a.lde; c += 2048) {
        const float f = vl_exp2(st[c >> 6].x - lse);
        bf16x8 v = *reinterpret_cast<const bf16x8*>(e + c);
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = f32_to_bf16(bf16_to_f32(v[k]) * f);
        *reinterpret_cast<bf16x8*>(e + c) = v;
    }
    __syncthreads();  // ... and every one is rewritten
#pragma unroll
    for (int i = 0; i < VL_MAX_TOP / 256; ++i)
        if ((mine >> i) & 1) e[tg.id[tid + i * 256]] = f32_to_bf16(val[i]);
}

// ---- on given logits: one workgroup per row
template <typename T>
struct Logits {
    const T* z;
    T* dz;                   // [rows][ldd], or nullptr
    long long ldz, ldd;
    const long long* ids;
    const float* p;
    const float* base;
    const int* valid;
    const float* scal;
    float* row_loss;
    int top, vocab;
    float scale_log2, inv_tau;
};

template <typename T>
__global__ __launch_bounds__(512) void logits_distill_kernel(const Logits<T> a) {
    __shared__ float red[16];
    __shared__ TargetLds tg;
    const int row = blockIdx.x, tid = threadIdx.x;
    const T* z = a.z + row * a.ldz;
    const bool valid = a.valid[row] != 0;
    T* dz = a.dz == nullptr ? nullptr : a.dz + row * a.ldd;
    if (!valid) {
        if (tid == 0) a.row_loss[row] = 0.f;
        if (dz != nullptr)
            for (int c = tid; c < a.vocab; c += 512) dz[c] = static_cast<T>(0.f);
        return;
    }
    vl_load_targets(tg, a.ids + static_cast<size_t>(row) * a.top, a.p + static_cast<size_t>(row) * a.top, a.top, a.vocab);
    float m = -VL_INF;
    for (int c = tid; c < a.vocab; c += 512) m = fmaxf(m, static_cast<float>(z[c]));
    m = block_max(m, red);
    const float ref = m == -VL_INF ? 0.f : m;
    float s = 0.f;
    for (int c = tid; c < a.vocab; c += 512) s += vl_exp2((static_cast<float>(z[c]) - ref) * a.scale_log2);
    s = block_sum(s, red);
    float t = 0.f;
    for (int k = tid; k < a.top; k += 512)
        if (tg.id[k] >= 0 && tg.p[k] != 0.f) t += tg.p[k] * (static_cast<float>(z[tg.id[k]]) - ref);
    t = block_sum(t, red);
    const float ls = log2f(s);
    if (tid == 0) a.row_loss[row] = a.base[row] - t * a.inv_tau + ls * VL_LN2;
    if (dz == nullptr) return;
    const float g = a.scal[0];
    auto q_of = [&](int c) { return vl_exp2((static_cast<float>(z[c]) - ref) * a.scale_log2 - ls); };
    for (int c = tid; c < a.vocab; c += 512) dz[c] = static_cast<T>(q_of(c) * g);
    __syncthreads();
    for (int k = tid; k < a.top; k += 512) {
        float p;
        if (vl_merged(tg, k, a.top, p)) dz[tg.id[k]] = static_cast<T>((q_of(tg.id[k]) - p) * g);
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

template <int KIND>
static int vl_launch(VocabGemm& g, int splits, hipStream_t s) {
    static unsigned long long granted;
    constexpr int lds = 2 * 2 * 256 * 64 * 2;
    if (int e = vl_grant_lds(vocab_gemm_kernel<KIND>, lds, granted)) return e;
    g.tiles_m = pdt_cdiv(g.M, 256);
    g.tiles_n = pdt_cdiv(g.N, 256);
    const long long blocks = static_cast<long long>(g.tiles_m) * g.tiles_n * splits;
    if (blocks >= (1ll << 31)) return -1;
    hipLaunchKernelGGL(vocab_gemm_kernel<KIND>, dim3(static_cast<unsigned>(blocks)), dim3(512), lds, s, g);
    return pdt_launch_status();
}

// Scores of `rows` rows against the vocabulary: stats [rows][ceil(vocab / 64)] {max, sum}; e [rows][lde] or nullptr, lde the
// vocabulary rounded up to 64.
PDT_API int pdt_vocab_scores(const void* x, const void* w, void* stats, void* e, int rows, int vocab, int width, long long lde, float inv_tau,
                             void* stream) {
    if (rows <= 0 || vocab <= 0 || width <= 0 || (width % 64) != 0 || (e != nullptr && lde != (vocab + 63ll) / 64 * 64) || !(inv_tau > 0.f)) return -1;
    VocabGemm g = {};
    g.a = static_cast<const bf16*>(x);
    g.b = static_cast<const bf16*>(w);
    g.lda = g.ldb = width;
    g.M = rows; g.N = vocab; g.K = g.k_per_split = width;
    g.stats = static_cast<float2*>(stats);
    g.e = static_cast<bf16*>(e);
    g.lde = lde;
    g.groups = pdt_cdiv(vocab, 64);
    g.scale_log2 = VL_LOG2E * inv_tau;
    return vl_launch<0>(g, 1, static_cast<hipStream_t>(stream));
}

PDT_API int pdt_vocab_targets(const long long* ids, const float* teacher, float* p, float* base, int* valid, float* scal, const void* x, const void* w,
                              void* x_used, int rows, int top, int width, int vocab, float tau, void* stream) {
    if (rows <= 0 || top <= 0 || top > VL_MAX_TOP || vocab <= 0 || !(tau > 0.f) || (x != nullptr && (width <= 0 || (width % 8) != 0))) return -1;
    if (teacher == nullptr && top != 1) return -1;
    hipStream_t s = static_cast<hipStream_t>(stream);
    Targets t = {ids, teacher, p, base, valid, static_cast<const bf16*>(x), static_cast<const bf16*>(w), static_cast<bf16*>(x_used), rows, top, width, vocab, 1.f / tau};
    hipLaunchKernelGGL(vocab_targets_kernel, dim3(pdt_cdiv(rows, 4)), dim3(256), 0, s, t);
    hipLaunchKernelGGL(vocab_count_kernel, dim3(1), dim3(1024), 0, s, valid, rows, tau, scal);
    return pdt_launch_status();
}

PDT_API int pdt_vocab_rows(const void* stats, void* e, const long long* ids, const float* p, const float* base, const int* valid, float* row_loss,
                           int rows, int vocab, int top, long long lde, void* stream) {
    if (rows <= 0 || vocab <= 0 || top <= 0 || top > VL_MAX_TOP) return -1;
    Rows a = {static_cast<const float2*>(stats), static_cast<bf16*>(e), lde, ids, p, base, valid, row_loss, pdt_cdiv(vocab, 64), top, vocab};
    hipLaunchKernelGGL(vocab_rows_kernel, dim3(rows), dim3(256), 0, static_cast<hipStream_t>(stream), a);
    return pdt_launch_status();
}

PDT_API int pdt_vocab_mean(const float* row_loss, const float* scal, float* loss, int rows, void* stream) {
    if (rows <= 0) return -1;
    hipLaunchKernelGGL(vocab_mean_kernel, dim3(1), dim3(1024), 0, static_cast<hipStream_t>(stream), row_loss, rows, scal, loss);
    return pdt_launch_status();
}

// Into how many parts the vocabulary is split for dx (1: no partial sums), so that few row tiles still fill the CUs.
PDT_API int pdt_vocab_dx_splits(int rows, int vocab, int width) {
    const int tiles = pdt_cdiv(rows, 256) * pdt_cdiv(width, 256), steps = pdt_cdiv(vocab, 64);
    int s = 256 / tiles;
    if (s > steps / 8) s = steps / 8;
    return s < 1 ? 1 : s;
}

// dx [rows][width] bf16 = scal[0] * D w.  part: splits * rows * width floats, unused where splits is 1.
PDT_API int pdt_vocab_dx(const void* d, const void* w, void* dx, float* part, int splits, const float* scal, int rows, int vocab, int width,
                         long long ldd, void* stream) {
    if (rows <= 0 || vocab <= 0 || width <= 0 || (width % 64) != 0 || ldd != (vocab + 63ll) / 64 * 64 || splits < 1 || (splits > 1 && part == nullptr))
        return -1;
    hipStream_t s = static_cast<hipStream_t>(stream);
    VocabGemm g = {};
    g.a = static_cast<const bf16*>(d);
    g.b = static_cast<const bf16*>(w);
    g.lda = ldd; g.ldb = width;
    g.M = rows; g.N = width; g.K = vocab;
    g.k_per_split = pdt_cdiv(pdt_cdiv(vocab, 64), splits) * 64;
    g.alpha = scal;
    g.ldo = width;
    if (splits > 1) g.out32 = part;
    else g.out = static_cast<bf16*>(dx);
    if (int e = vl_launch<1>(g, splits, s)) return e;
    if (splits > 1) {
        const long long n = static_cast<long long>(rows) * width, blocks = (n / 4 + 255) / 256;
        hipLaunchKernelGGL(vocab_join_kernel, dim3(static_cast<unsigned>(blocks < 4096 ? blocks : 4096)), dim3(256), 0, s, part, splits, n, scal,
                           static_cast<bf16*>(dx));
    }
    return pdt_launch_status();
}

// dw [vocab][width] = scal[0] * D^T x, bf16 (dw) or fp32 (dw32, added to what it holds if accumulate)
PDT_API int pdt_vocab_dw(const void* d, const void* x, void* dw, float* dw32, int accumulate, const float* scal, const void* zeros, int rows, int vocab,
                         int width, long long ldd, void* stream) {
    if (rows <= 0 || vocab <= 0 || width <= 0 || (width % 64) != 0 || ldd != (vocab + 63ll) / 64 * 64 || (dw == nullptr) == (dw32 == nullptr) ||
        zeros == nullptr)
        return -1;
    VocabGemm g = {};
    g.a = static_cast<const bf16*>(d);
    g.b = static_cast<const bf16*>(x);
    g.lda = ldd; g.ldb = width;
    g.M = vocab; g.N = width; g.K = rows;
    g.k_per_split = (rows + 63) / 64 * 64;
    g.zeros = static_cast<const bf16*>(zeros);
    g.alpha = scal;
    g.out = static_cast<bf16*>(dw);
    g.out32 = dw32;
    g.accumulate = accumulate;
    g.ldo = width;
    return vl_launch<2>(g, 1, static_cast<hipStream_t>(stream));
}

// dtype: 0 fp32, 1 bf16 logits.  dz (may be nullptr) has the logits' type and row pitch ldd.
PDT_API int pdt_logits_distill(const void* z, void* dz, const long long* ids, const float* p, const float* base, const int* valid, const float* scal,
                               float* row_loss, int rows, int vocab, int top, long long ldz, long long ldd, float inv_tau, int dtype, void* stream) {
    if (rows <= 0 || vocab <= 0 || top <= 0 || top > VL_MAX_TOP || ldz < 0 || (dz != nullptr && ldd < vocab) || !(inv_tau > 0.f)) return -1;
    hipStream_t s = static_cast<hipStream_t>(stream);
    const float c = VL_LOG2E * inv_tau;
    if (dtype == 1) {
        Logits<bf16> a = {static_cast<const bf16*>(z), static_cast<bf16*>(dz), ldz, ldd, ids, p, base, valid, scal, row_loss, top, vocab, c, inv_tau};
        hipLaunchKernelGGL(logits_distill_kernel<bf16>, dim3(rows), dim3(512), 0, s, a);
    } else {
        Logits<float> a = {static_cast<const float*>(z), static_cast<float*>(dz), ldz, ldd, ids, p, base, valid, scal, row_loss, top, vocab, c, inv_tau};
        hipLaunchKernelGGL(logits_distill_kernel<float>, dim3(rows), dim3(512), 0, s, a);
    }
    return pdt_launch_status();
}
