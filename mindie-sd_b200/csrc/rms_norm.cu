// Residual addition, root-mean-square norm and per-token e4m3 quantisation of [rows, dim] activations.
//
//   v = x + residual,  rstd = 1 / sqrt(mean(v^2) + eps),  y = (v * w) * rstd          (all in fp32)
//   out = y in the type of x, or e4m3 of y / scale with scale = max|y| / 448 per row
//   residual_out = v, rounded once to the residual's type
//
// Bound by HBM: a row is read once, kept in registers as fp32 between the reduction and the stores, and
// written once.  max|y| = max|v w| * rstd holds exactly in fp32 (a product with one positive factor keeps
// the order of rounded products), so the sum of squares and the maximum come out of ONE reduction and the
// quantised form costs no second one.
#include "capi_common.h"
#include "row_io.cuh"

namespace sdb {
namespace {

constexpr float kE4m3Max = 448.0f;
constexpr float kMinScale = 1.17549435e-38f;  // 2^-126: below it 1 / scale would overflow

struct NormParams {
    const void* x;
    const void* residual;  // or null
    const void* weight;    // or null
    void* out;
    void* residual_out;
    float* scales;  // not null: out is e4m3
    int64_t rows, x_stride, residual_stride;
    int dim;
    int residual_fp32, weight_fp32;  // else the type of x
    int norm;                        // 0: y = v (quantiser alone)
    int group;                       // threads per row, a power of two
    float eps, inv_dim;
};

struct Stats {
    float sum, top;
};

// Combines the statistics of the `group` threads of a row.  Up to a warp by shuffles; beyond that the
// block holds one row and the warps meet in shared memory, every thread adding the partials in one order.
__device__ __forceinline__ Stats reduce_row(Stats s, int group) {
    const int width = group < 32 ? group : 32;
    for (int d = width >> 1; d > 0; d >>= 1) {
        s.sum += __shfl_xor_sync(0xffffffffu, s.sum, d);
        s.top = max_nan(s.top, __shfl_xor_sync(0xffffffffu, s.top, d));
    }
    if (group > 32) {
        __shared__ Stats part[32];
        if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = s;
        __syncthreads();
        s = part[(threadIdx.x & ~(group - 1)) >> 5];
        const int first = (threadIdx.x & ~(group - 1)) >> 5;
        for (int i = 1; i < (group >> 5); ++i) {
            s.sum += part[first + i].sum;
            s.top = max_nan(s.top, part[first + i].top);
        }
    }
    return s;
}

// Factors that turn v * w into the stored value, from the row's statistics.
__device__ __forceinline__ float row_factor(const NormParams& p, const Stats& s, float& scale) {
    const float rstd = p.norm ? rsqrtf(s.sum * p.inv_dim + p.eps) : 1.0f;
    if (!p.scales) return rstd;
    const float top = s.top * rstd;
    scale = top == 0.0f ? 1.0f : max_nan(top / kE4m3Max, kMinScale);
    return rstd * (1.0f / scale);
}

template <typename T, int kE>
__device__ __forceinline__ void store_run(const NormParams& p, int64_t at, const float (&y)[kE]) {
    if (p.scales) {
        uint8_t* o = static_cast<uint8_t*>(p.out) + at;
        if constexpr (kE == 1) {
            *o = static_cast<uint8_t>(e4m3x2(y[0], 0.0f) & 0xff);
        } else {
            union {
                uint16_t h[kE / 2];
                typename Raw<kE>::type raw;
            } u;
#pragma unroll
            for (int i = 0; i < kE / 2; ++i) u.h[i] = e4m3x2(y[2 * i], y[2 * i + 1]);
            *reinterpret_cast<typename Raw<kE>::type*>(o) = u.raw;
        }
    } else {
        Run<T, kE> r;
#pragma unroll
        for (int i = 0; i < kE; ++i) r.set(i, y[i]);
        r.store(static_cast<T*>(p.out) + at);
    }
}

template <typename T, int kE>
__device__ __forceinline__ void weights_of(const NormParams& p, int at, float (&w)[kE]) {
    if (!p.weight) {
#pragma unroll
        for (int i = 0; i < kE; ++i) w[i] = 1.0f;
    } else if (p.weight_fp32) {
        Run<float, kE> r;
        r.load(static_cast<const float*>(p.weight) + at);
#pragma unroll
        for (int i = 0; i < kE; ++i) w[i] = r.get(i);
    } else {
        Run<T, kE> r;
        r.load(static_cast<const T*>(p.weight) + at);
#pragma unroll
        for (int i = 0; i < kE; ++i) w[i] = r.get(i);
    }
}

// One row per `group` threads, kV runs of kE elements per thread, the row in registers.  Runs of 16 bytes
// where every row starts on such a boundary, 8 bytes or single elements where only that holds.
template <typename T, int kE, int kV>
__global__ void __launch_bounds__(1024) norm_row_kernel(const NormParams p) {
    const int lane = threadIdx.x & (p.group - 1);
    const int64_t row = static_cast<int64_t>(blockIdx.x) * (blockDim.x / p.group) + threadIdx.x / p.group;
    const bool live = row < p.rows;  // the threads of a missing row still take part in the shuffles
    const T* x = static_cast<const T*>(p.x) + row * p.x_stride;
    float v[kV][kE];
    {
        Run<T, kE> in[kV];
#pragma unroll
        for (int j = 0; j < kV; ++j) {
            const int at = (lane + j * p.group) * kE;
            if (live && at < p.dim) in[j].load(x + at);
        }
        if (p.residual && p.residual_fp32) {
            const float* r = static_cast<const float*>(p.residual) + row * p.residual_stride;
            Run<float, kE> add[kV];
#pragma unroll
            for (int j = 0; j < kV; ++j) {
                const int at = (lane + j * p.group) * kE;
                if (live && at < p.dim) add[j].load(r + at);
            }
#pragma unroll
            for (int j = 0; j < kV; ++j)
#pragma unroll
                for (int i = 0; i < kE; ++i) v[j][i] = in[j].get(i) + add[j].get(i);
        } else if (p.residual) {
            const T* r = static_cast<const T*>(p.residual) + row * p.residual_stride;
            Run<T, kE> add[kV];
#pragma unroll
            for (int j = 0; j < kV; ++j) {
                const int at = (lane + j * p.group) * kE;
                if (live && at < p.dim) add[j].load(r + at);
            }
#pragma unroll
            for (int j = 0; j < kV; ++j)
#pragma unroll
                for (int i = 0; i < kE; ++i) v[j][i] = in[j].get(i) + add[j].get(i);
        } else {
#pragma unroll
            for (int j = 0; j < kV; ++j)
#pragma unroll
                for (int i = 0; i < kE; ++i) v[j][i] = in[j].get(i);
        }
    }
    Stats s = {0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < kV; ++j) {
        const int at = (lane + j * p.group) * kE;
        if (!live || at >= p.dim) continue;
        if (p.residual) {
            const int64_t o = row * p.dim + at;
            if (p.residual_fp32) {
                Run<float, kE> r;
#pragma unroll
                for (int i = 0; i < kE; ++i) r.set(i, v[j][i]);
                r.store(static_cast<float*>(p.residual_out) + o);
            } else {
                Run<T, kE> r;
#pragma unroll
                for (int i = 0; i < kE; ++i) r.set(i, v[j][i]);
                r.store(static_cast<T*>(p.residual_out) + o);
            }
        }
        float w[kE];
        weights_of<T, kE>(p, at, w);
#pragma unroll
        for (int i = 0; i < kE; ++i) {
            s.sum += v[j][i] * v[j][i];
            v[j][i] *= w[i];
            s.top = max_nan(s.top, fabsf(v[j][i]));
        }
    }
    s = reduce_row(s, p.group);
    float scale = 1.0f;
    const float f = row_factor(p, s, scale);
    if (!live) return;
    if (p.scales && lane == 0) p.scales[row] = scale;
#pragma unroll
    for (int j = 0; j < kV; ++j) {
        const int at = (lane + j * p.group) * kE;
        if (at >= p.dim) continue;
#pragma unroll
        for (int i = 0; i < kE; ++i) v[j][i] *= f;
        store_run<T, kE>(p, row * p.dim + at, v[j]);
    }
}

// Rows too long for the registers of a block: one block per row, the row read twice (the second time from L2).
template <typename T>
__global__ void __launch_bounds__(1024) norm_long_kernel(const NormParams p) {
    const int64_t row = blockIdx.x;
    const T* x = static_cast<const T*>(p.x) + row * p.x_stride;
    auto value = [&](int at) {
        float v = to_f32(x[at]);
        if (p.residual) {
            const int64_t r = row * p.residual_stride + at;
            v += p.residual_fp32 ? static_cast<const float*>(p.residual)[r] : to_f32(static_cast<const T*>(p.residual)[r]);
        }
        return v;
    };
    auto weight = [&](int at) {
        if (!p.weight) return 1.0f;
        return p.weight_fp32 ? static_cast<const float*>(p.weight)[at] : to_f32(static_cast<const T*>(p.weight)[at]);
    };
    Stats s = {0.0f, 0.0f};
    for (int at = threadIdx.x; at < p.dim; at += blockDim.x) {
        const float v = value(at);
        if (p.residual) {
            const int64_t o = row * p.dim + at;
            if (p.residual_fp32) static_cast<float*>(p.residual_out)[o] = v;
            else static_cast<T*>(p.residual_out)[o] = from_f32<T>(v);
        }
        s.sum += v * v;
        s.top = max_nan(s.top, fabsf(v * weight(at)));
    }
    s = reduce_row(s, p.group);
    float scale = 1.0f;
    const float f = row_factor(p, s, scale);
    if (p.scales && threadIdx.x == 0) p.scales[row] = scale;
    for (int at = threadIdx.x; at < p.dim; at += blockDim.x) {
        const float y[1] = {value(at) * weight(at) * f};
        store_run<T, 1>(p, row * p.dim + at, y);
    }
}

template <typename T, int kE>
cudaError_t launch_rows(NormParams p, cudaStream_t stream) {
    const int runs = (p.dim + kE - 1) / kE;
    // The smallest group of threads that holds the row in at most kMaxRuns runs each.
    constexpr int kMaxRuns = 6;
    int group = 1;
    while (group < 1024 && group * kMaxRuns < runs) group *= 2;
    const int per_thread = (runs + group - 1) / group;
    if (per_thread > kMaxRuns) {
        p.group = 1024;
        norm_long_kernel<T><<<static_cast<unsigned>(p.rows), 1024, 0, stream>>>(p);
        return cudaGetLastError();
    }
    p.group = group;
    const int threads = group > 128 ? group : 128;
    const int64_t blocks = (p.rows + threads / group - 1) / (threads / group);
    const unsigned grid = static_cast<unsigned>(blocks);
    switch (per_thread) {
        case 1: norm_row_kernel<T, kE, 1><<<grid, threads, 0, stream>>>(p); break;
        case 2: norm_row_kernel<T, kE, 2><<<grid, threads, 0, stream>>>(p); break;
        case 3: norm_row_kernel<T, kE, 3><<<grid, threads, 0, stream>>>(p); break;
        case 4: norm_row_kernel<T, kE, 4><<<grid, threads, 0, stream>>>(p); break;
        case 5: norm_row_kernel<T, kE, 5><<<grid, threads, 0, stream>>>(p); break;
        default: norm_row_kernel<T, kE, 6><<<grid, threads, 0, stream>>>(p); break;
    }
    return cudaGetLastError();
}

// The widest run that every row of every operand starts on.
template <typename T>
cudaError_t launch_typed(const NormParams& p, cudaStream_t stream) {
    auto rows_at = [](const void* base, int64_t stride, int elem, int run) {
        const int bytes = elem * run < 16 ? elem * run : 16;
        return !base || (reinterpret_cast<uintptr_t>(base) % bytes == 0 && (stride * elem) % bytes == 0);
    };
    const int e = static_cast<int>(sizeof(T));
    auto fits = [&](int run) {
        const int re = p.residual_fp32 ? 4 : e, oe = p.scales ? 1 : e;
        return p.dim % run == 0 && rows_at(p.x, p.x_stride, e, run) && rows_at(p.residual, p.residual_stride, re, run) &&
               rows_at(p.residual_out, p.dim, re, run) && rows_at(p.weight, 0, p.weight_fp32 ? 4 : e, run) &&
               rows_at(p.out, p.dim, oe, run);
    };
    if constexpr (sizeof(T) == 2) {
        if (fits(8)) return launch_rows<T, 8>(p, stream);
    }
    if (fits(4)) return launch_rows<T, 4>(p, stream);
    return launch_rows<T, 1>(p, stream);
}

}  // namespace
}  // namespace sdb

using namespace sdb;

extern "C" int mindiesd_add_rms_norm(const mindiesd_norm_args* a, void* stream_) {
    if (!a || !a->x || !a->out) return MINDIESD_E_NULL;
    if ((a->residual == nullptr) != (a->residual_out == nullptr)) return MINDIESD_E_NULL;
    if (a->rows <= 0 || a->rows > 0x7fffffff || a->dim <= 0) return MINDIESD_E_SHAPE;
    if (a->dtype != MINDIESD_BF16 && a->dtype != MINDIESD_FP16 && a->dtype != MINDIESD_FP32) return MINDIESD_E_DTYPE;
    if (a->residual && a->residual_dtype != a->dtype && a->residual_dtype != MINDIESD_FP32) return MINDIESD_E_DTYPE;
    if (a->weight && a->weight_dtype != a->dtype && a->weight_dtype != MINDIESD_FP32) return MINDIESD_E_DTYPE;
    if (a->out_dtype == MINDIESD_E4M3) {
        if (!a->scales) return MINDIESD_E_NULL;
    } else if (a->out_dtype != a->dtype) {
        return MINDIESD_E_DTYPE;
    }
    if (a->x_stride < 0 || (a->residual && a->residual_stride < 0)) return MINDIESD_E_STRIDE;
    const int e = dtype_bytes(a->dtype);
    auto aligned = [](const void* ptr, int bytes) { return reinterpret_cast<uintptr_t>(ptr) % bytes == 0; };
    if (!aligned(a->x, e) || !aligned(a->out, dtype_bytes(a->out_dtype)) || !aligned(a->scales, 4)) return MINDIESD_E_STRIDE;
    if (a->residual && (!aligned(a->residual, dtype_bytes(a->residual_dtype)) ||
                        !aligned(a->residual_out, dtype_bytes(a->residual_dtype))))
        return MINDIESD_E_STRIDE;
    if (a->weight && !aligned(a->weight, dtype_bytes(a->weight_dtype))) return MINDIESD_E_STRIDE;
    if (!a->quant_only && !(a->eps > 0.0f && a->eps < 1e30f)) return MINDIESD_E_VALUE;
    if (a->quant_only && (a->weight || a->residual || a->out_dtype != MINDIESD_E4M3)) return MINDIESD_E_VALUE;
    NormParams p = {};
    p.x = a->x;
    p.residual = a->residual;
    p.weight = a->weight;
    p.out = a->out;
    p.residual_out = a->residual_out;
    p.scales = a->out_dtype == MINDIESD_E4M3 ? a->scales : nullptr;
    p.rows = a->rows;
    p.dim = a->dim;
    p.x_stride = a->x_stride;
    p.residual_stride = a->residual_stride;
    p.residual_fp32 = a->residual && a->residual_dtype == MINDIESD_FP32;
    p.weight_fp32 = a->weight && a->weight_dtype == MINDIESD_FP32;
    p.norm = a->quant_only ? 0 : 1;
    p.eps = a->eps;
    p.inv_dim = 1.0f / static_cast<float>(a->dim);
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    cudaError_t err;
    if (a->dtype == MINDIESD_BF16) err = launch_typed<__nv_bfloat16>(p, stream);
    else if (a->dtype == MINDIESD_FP16) err = launch_typed<__half>(p, stream);
    else err = launch_typed<float>(p, stream);
    return err == cudaSuccess ? MINDIESD_OK : static_cast<int>(err);
}
