// Fused softmax cross-entropy for bf16 or fp32 logits, mean over the rows whose label is one of the classes: a label outside
// (-100, say) leaves its row out, without gradient and not counted; 0 where no row has one.
//
// Forward: one pass per row computes max, log-sum-exp and the row loss (online softmax, so the
//          row is read once even when it does not fit in registers); the row's lse is kept.
// Backward: dlogits = (exp(x - lse) - onehot) * (g / rows with a label), written in the logits' dtype in
//          one pass; probabilities are never materialised.
// Rows of up to 1024 classes are handled by one wave each (4 rows per workgroup); longer rows
// (language-model vocabularies) by one 256-thread workgroup each.
//
// Role parity: nn.CrossEntropyLoss (log_softmax + nll_loss, mean reduction) at
// /root/reference/src/main.py:62,76,78.
#include "common.h"

template <typename T>
__device__ __forceinline__ float ld(const T* p, long long i);
template <>
__device__ __forceinline__ float ld<bf16>(const bf16* p, long long i) { return bf16_to_f32(p[i]); }
template <>
__device__ __forceinline__ float ld<float>(const float* p, long long i) { return p[i]; }

template <typename T>
__device__ __forceinline__ void st(T* p, long long i, float v);
template <>
__device__ __forceinline__ void st<bf16>(bf16* p, long long i, float v) { p[i] = f32_to_bf16(v); }
template <>
__device__ __forceinline__ void st<float>(float* p, long long i, float v) { p[i] = v; }

// Running-max sentinel: finite, so exp(m - m) is 1 (not NaN) when two empty partials are merged and
// the code stays correct under -ffast-math (which assumes no infinities).
#define CE_NEG (-3.0e38f)

__device__ __forceinline__ void online_merge(float& m, float& s, float m2, float s2) {
    const float mn = fmaxf(m, m2);
    s = s * __expf(m - mn) + s2 * __expf(m2 - mn);
    m = mn;
}

// rows with a label, 1 where there are none (the sums they divide are 0 then)
__device__ __forceinline__ float label_count(const long long* __restrict__ labels, long long rows, int classes, float* red) {
    float c = 0.f;
    for (long long i = threadIdx.x; i < rows; i += blockDim.x) c += labels[i] >= 0 && labels[i] < classes ? 1.f : 0.f;
    return fmaxf(block_sum(c, red), 1.f);  // (whole numbers: exact up to 2^24 rows, and every thread's share far below)
}
__global__ __launch_bounds__(1024) void label_count_kernel(const long long* __restrict__ labels, long long rows, int classes, float* __restrict__ count) {
    __shared__ float red[16];
    const float c = label_count(labels, rows, classes, red);
    if (threadIdx.x == 0) count[0] = c;
}

// ---- wave-per-row forward
template <typename T>
__global__ __launch_bounds__(256) void ce_fwd_wave_kernel(const T* __restrict__ logits, const long long* __restrict__ labels,
                                                         float* __restrict__ row_loss, float* __restrict__ lse, int rows,
                                                         int classes, long long ld_row) {
    const int lane = threadIdx.x & 63;
    const int row = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= rows) return;
    const T* x = logits + row * ld_row;
    float m = CE_NEG, s = 0.f;
    for (int i = lane; i < classes; i += 64) {
        const float v = ld<T>(x, i);
        const float mn = fmaxf(m, v);
        s = s * __expf(m - mn) + __expf(v - mn);
        m = mn;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const float m2 = __shfl_xor(m, o, 64), s2 = __shfl_xor(s, o, 64);
        online_merge(m, s, m2, s2);
    }
    if (lane == 0) {
        const float l = m + __logf(s);
        const long long y = labels[row];
        lse[row] = l;
        row_loss[row] = (y >= 0 && y < classes) ? l - ld<T>(x, y) : 0.f;
    }
}

// ---- workgroup-per-row forward (long rows)
template <typename T>
__global__ __launch_bounds__(256) void ce_fwd_block_kernel(const T* __restrict__ logits, const long long* __restrict__ labels,
                                                          float* __restrict__ row_loss, float* __restrict__ lse,
                                                          int classes, long long ld_row) {
    __shared__ float sm[4], ss[4];
    const int row = blockIdx.x;
    const T* x = logits + row * ld_row;
    float m = CE_NEG, s = 0.f;
    for (int i = threadIdx.x; i < classes; i += 256) {
        const float v = ld<T>(x, i);
        const float mn = fmaxf(m, v);
        s = s * __expf(m - mn) + __expf(v - mn);
        m = mn;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const float m2 = __shfl_xor(m, o, 64), s2 = __shfl_xor(s, o, 64);
        online_merge(m, s, m2, s2);
    }
    if ((threadIdx.x & 63) == 0) {
        sm[threadIdx.x >> 6] = m;
        ss[threadIdx.x >> 6] = s;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        float M = sm[0], S = ss[0];
        for (int w = 1; w < 4; ++w)
            online_merge(M, S, sm[w], ss[w]);
        const float l = M + __logf(S);
        const long long y = labels[row];
        lse[row] = l;
        row_loss[row] = (y >= 0 && y < classes) ? l - ld<T>(x, y) : 0.f;
    }
}

// ---- backward: grid-stride over all elements of the [rows, classes] matrix
template <typename T>
__global__ __launch_bounds__(256) void ce_bwd_kernel(const T* __restrict__ logits, const long long* __restrict__ labels,
                                                    const float* __restrict__ lse, const float* __restrict__ gout,
                                                    const float* __restrict__ count, T* __restrict__ dlogits, int rows,
                                                    int classes, long long ld_row, long long ld_drow, int pad_to) {
    const float g = gout[0] / count[0];
    // one workgroup walks whole rows so lse/label are loaded once per row
    for (int row = blockIdx.x; row < rows; row += gridDim.x) {
        const float l = lse[row];
        const long long y = labels[row];
        const T* x = logits + row * ld_row;
        T* d = dlogits + row * ld_drow;
        const bool valid = y >= 0 && y < classes;
        for (int i = threadIdx.x; i < pad_to; i += 256) {
            float v = 0.f;
            if (i < classes && valid) v = (__expf(ld<T>(x, i) - l) - (i == y ? 1.f : 0.f)) * g;
            st<T>(d, i, v);
        }
    }
}

// ---- long bf16 rows, forward and gradient in one pass: a 512-thread workgroup holds its row in registers
// (NV 16-byte vectors per thread), so the logits are read from memory once and the gradient
// (softmax - onehot) / (rows with a label) is written straight away; the backward pass only has to scale it by the
// incoming gradient, which for a loss that is the root of the graph is 1.
template <int NV>
__global__ __launch_bounds__(512) void ce_fused_row_kernel(const bf16* __restrict__ logits, const long long* __restrict__ labels,
                                                          float* __restrict__ row_loss, bf16* __restrict__ dlogits,
                                                          int rows, int classes, long long ld_row, long long ld_drow,
                                                          int pad_to, const float* __restrict__ count) {
    __shared__ float red[16];
    const int row = blockIdx.x;
    const bf16* x = logits + row * ld_row;
    const int nvec = (classes + 7) >> 3;  // vectors that hold at least one class (ld_row covers them)
    bf16x8 v[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int vi = threadIdx.x + i * 512;
        if (vi < nvec) v[i] = *reinterpret_cast<const bf16x8*>(x + vi * 8);
    }
    const long long y = labels[row];
    const bool valid = y >= 0 && y < classes;
    float m = CE_NEG, xy = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int vi = threadIdx.x + i * 512;
        if (vi < nvec) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int c = vi * 8 + e;
                const float f = bf16_to_f32(v[i][e]);
                if (c < classes) m = fmaxf(m, f);
                if (c == y) xy = f;
            }
        }
    }
    m = block_max(m, red);
    const float ml2 = m * 1.4426950408889634f;
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int vi = threadIdx.x + i * 512;
        if (vi < nvec) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (vi * 8 + e < classes) s += __builtin_amdgcn_exp2f(bf16_to_f32(v[i][e]) * 1.4426950408889634f - ml2);
        }
    }
    s = block_sum(s, red);
    xy = block_sum(xy, red);  // one thread holds the label's logit, the others 0
    const float l = m + __logf(s);
    if (threadIdx.x == 0) row_loss[row] = valid ? l - xy : 0.f;
    if (dlogits == nullptr) return;
    // (dlogits may be the logits buffer itself: every thread has its part of the row in registers by now, and the
    // block reductions above are barriers between the last load and the first store)
    const float g = valid ? 1.f / count[0] : 0.f;
    const float ll2 = l * 1.4426950408889634f;
    bf16* d = dlogits + row * ld_drow;
    const int pvec = pad_to >> 3;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int vi = threadIdx.x + i * 512;
        if (vi < pvec) {
            bf16x8 o;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int c = vi * 8 + e;
                float r = 0.f;
                if (vi < nvec && c < classes && valid)
                    r = (__builtin_amdgcn_exp2f(bf16_to_f32(v[i][e]) * 1.4426950408889634f - ll2) - (c == y ? 1.f : 0.f)) * g;
                o[e] = f32_to_bf16(r);
            }
            *reinterpret_cast<bf16x8*>(d + vi * 8) = o;
        }
    }
}

// x *= g[0] unless g[0] == 1 (the gradient of a loss that is the root of the graph)
__global__ __launch_bounds__(256) void scale_by_scalar_kernel(bf16* __restrict__ x, const float* __restrict__ g, long long nvec) {
    const float gv = g[0];
    if (gv == 1.f) return;
    for (long long i = blockIdx.x * 256ll + threadIdx.x; i < nvec; i += gridDim.x * 256ll) {
        bf16x8 v = *reinterpret_cast<bf16x8*>(x + i * 8);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = f32_to_bf16(bf16_to_f32(v[e]) * gv);
        *reinterpret_cast<bf16x8*>(x + i * 8) = v;
    }
}

// Sum of the row losses over the rows with a label (single workgroup, fixed order): counted from the labels and left in
// count, or - where labels is nullptr - as count says.
__global__ __launch_bounds__(1024) void ce_mean_kernel(const float* __restrict__ row_loss, const long long* __restrict__ labels, long long rows,
                                                      int classes, float* __restrict__ count, float* __restrict__ loss) {
    __shared__ float red[16];
    float s = 0.f;
    for (long long i = threadIdx.x; i < rows; i += 1024) s += row_loss[i];
    const float t = block_sum(s, red);
    const float c = labels != nullptr ? label_count(labels, rows, classes, red) : count[0];
    if (threadIdx.x == 0) {
        loss[0] = t * (1.f / c);
        if (labels != nullptr) count[0] = c;
    }
}

// dtype: 0 = fp32 logits, 1 = bf16 logits.  row_loss/lse: [rows] fp32.  loss: [1] fp32.  count: [1] fp32,
// the rows with a label (at least 1), for the backward pass.
PDT_API int pdt_softmax_ce_fwd(const void* logits, const long long* labels, float* row_loss, float* lse, float* loss, float* count,
                               int rows, int classes, long long ld_row, int dtype, void* stream) {
    if (rows <= 0 || classes <= 0 || ld_row < classes) return -1;
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (classes <= 1024) {
        const dim3 g(pdt_cdiv(rows, 4)), b(256);
        if (dtype == 1) hipLaunchKernelGGL(ce_fwd_wave_kernel<bf16>, g, b, 0, s, static_cast<const bf16*>(logits), labels, row_loss, lse, rows, classes, ld_row);
        else hipLaunchKernelGGL(ce_fwd_wave_kernel<float>, g, b, 0, s, static_cast<const float*>(logits), labels, row_loss, lse, rows, classes, ld_row);
    } else {
        const dim3 g(rows), b(256);
        if (dtype == 1) hipLaunchKernelGGL(ce_fwd_block_kernel<bf16>, g, b, 0, s, static_cast<const bf16*>(logits), labels, row_loss, lse, classes, ld_row);
        else hipLaunchKernelGGL(ce_fwd_block_kernel<float>, g, b, 0, s, static_cast<const float*>(logits), labels, row_loss, lse, classes, ld_row);
    }
    hipLaunchKernelGGL(ce_mean_kernel, dim3(1), dim3(1024), 0, s, row_loss, labels, static_cast<long long>(rows), classes, count, loss);
    return pdt_launch_status();
}

// dlogits has row stride ld_drow; columns [classes, pad_to) are written as zeros (pad_to <= ld_drow).
PDT_API int pdt_softmax_ce_bwd(const void* logits, const long long* labels, const float* lse, const float* gout, const float* count,
                               void* dlogits, int rows, int classes, long long ld_row, long long ld_drow, int pad_to,
                               int dtype, void* stream) {
    if (rows <= 0 || classes <= 0 || ld_row < classes || pad_to < classes || ld_drow < pad_to) return -1;
    hipStream_t s = static_cast<hipStream_t>(stream);
    const dim3 g(rows < 8192 ? rows : 8192), b(256);
    if (dtype == 1) hipLaunchKernelGGL(ce_bwd_kernel<bf16>, g, b, 0, s, static_cast<const bf16*>(logits), labels, lse, gout, count, static_cast<bf16*>(dlogits), rows, classes, ld_row, ld_drow, pad_to);
    else hipLaunchKernelGGL(ce_bwd_kernel<float>, g, b, 0, s, static_cast<const float*>(logits), labels, lse, gout, count, static_cast<float*>(dlogits), rows, classes, ld_row, ld_drow, pad_to);
    return pdt_launch_status();
}

// Forward and gradient in one pass for bf16 logits with long rows (see ce_fused_row_kernel): row losses and the logits'
// gradient for an incoming one of 1 (scale with pdt_scale_by_scalar), of a batch of which count[0] rows have a label
// (pdt_label_count); pdt_label_mean takes the mean.  A batch may come in chunks of rows.  dlogits may be nullptr (no gradient
// wanted) or the logits buffer itself: a language-model head then needs no second [rows, vocabulary] buffer; it has row stride
// ld_drow and columns [classes, pad_to) are written as zeros.  Needs classes > 1024, ld_row, ld_drow and pad_to multiples of
// 8, ld_row >= classes rounded up to 8, and at most 65536 classes.
PDT_API int pdt_softmax_ce_fused(const void* logits, const long long* labels, float* row_loss, void* dlogits, int rows, int classes,
                                 long long ld_row, long long ld_drow, int pad_to, const float* count, void* stream) {
    const int c8 = (classes + 7) / 8 * 8;
    if (rows <= 0 || classes <= 1024 || classes > 65536 || (ld_row % 8) != 0 || ld_row < c8) return -1;
    if (dlogits != nullptr && ((ld_drow % 8) != 0 || (pad_to % 8) != 0 || pad_to < c8 || ld_drow < pad_to || pad_to > 65536)) return -1;
    hipStream_t s = static_cast<hipStream_t>(stream);
    const int need = (((dlogits != nullptr ? pad_to : c8) >> 3) + 511) / 512;
    const bf16* x = static_cast<const bf16*>(logits);
    bf16* d = static_cast<bf16*>(dlogits);
#define PDT_CE(NV) hipLaunchKernelGGL(ce_fused_row_kernel<NV>, dim3(rows), dim3(512), 0, s, x, labels, row_loss, d, rows, classes, ld_row, ld_drow, pad_to, count)
    if (need <= 4) PDT_CE(4);
    else if (need <= 8) PDT_CE(8);
    else if (need <= 13) PDT_CE(13);
    else PDT_CE(16);
#undef PDT_CE
    return pdt_launch_status();
}

// count[0] = rows with a label, at least 1
PDT_API int pdt_label_count(const long long* labels, long long rows, int classes, float* count, void* stream) {
    if (rows <= 0 || classes <= 0) return -1;
    hipLaunchKernelGGL(label_count_kernel, dim3(1), dim3(1024), 0, static_cast<hipStream_t>(stream), labels, rows, classes, count);
    return pdt_launch_status();
}

// loss[0] = sum(row_loss) / count[0] (one workgroup, fixed order)
PDT_API int pdt_label_mean(const float* row_loss, long long rows, const float* count, float* loss, void* stream) {
    if (rows <= 0) return -1;
    hipLaunchKernelGGL(ce_mean_kernel, dim3(1), dim3(1024), 0, static_cast<hipStream_t>(stream), row_loss, nullptr, rows, 0, const_cast<float*>(count), loss);
    return pdt_launch_status();
}

// dst += g[0] * src over fp32 vectors (n a multiple of 4): a gradient computed for an incoming gradient of 1 is
// added to its destination once the incoming gradient is known
__global__ __launch_bounds__(256) void axpy_dev_scalar_kernel(float4* __restrict__ dst, const float4* __restrict__ src,
                                                              const float* __restrict__ g, long long n4) {
    const float gv = g[0];
    for (long long i = blockIdx.x * 256ll + threadIdx.x; i < n4; i += gridDim.x * 256ll) {
        float4 d = dst[i];
        const float4 a = src[i];
        d.x += gv * a.x;
        d.y += gv * a.y;
        d.z += gv * a.z;
        d.w += gv * a.w;
        dst[i] = d;
    }
}

PDT_API int pdt_axpy_dev_scalar_f32(float* dst, const float* src, const float* g, long long n, void* stream) {
    if (n <= 0 || (n % 4) != 0) return -1;
    long long blocks = (n / 4 + 255) / 256;
    if (blocks > 8192) blocks = 8192;
    hipLaunchKernelGGL(axpy_dev_scalar_kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, static_cast<hipStream_t>(stream),
                       reinterpret_cast<float4*>(dst), reinterpret_cast<const float4*>(src), g, n / 4);
    return pdt_launch_status();
}

PDT_API int pdt_scale_by_scalar(void* x, const float* g, long long numel, void* stream) {
    if (numel <= 0 || (numel % 8) != 0) return -1;
    long long blocks = (numel / 8 + 255) / 256;
    if (blocks > 4096) blocks = 4096;
    hipLaunchKernelGGL(scale_by_scalar_kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, static_cast<hipStream_t>(stream),
                       static_cast<bf16*>(x), g, numel / 8);
    return pdt_launch_status();
}
