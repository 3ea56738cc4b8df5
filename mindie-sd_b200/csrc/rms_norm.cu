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
#include "ptx_sm100.cuh"
#include "row_io.cuh"

#include <algorithm>
#include <atomic>
#include <type_traits>

namespace sdb {
namespace {

constexpr float kE4m3Max = 448.0f;
constexpr float kMinScale = 1.17549435e-38f;  // 2^-126: below it 1 / scale would overflow
constexpr float kMaxFloat = 3.40282347e38f;   // what is above it is infinite

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
    int residual_out32;              // rows of residual_out start on 32 bytes
    int norm;                        // 0: y = v (quantiser alone)
    int group;                       // threads per row, a power of two
    float eps, inv_dim;
};

struct Stats {
    float sum, top;
};

// Combines the statistics of the `group` threads of a row.  Up to a warp by shuffles; beyond that the
// block holds one row and the warps meet in shared memory, every thread adding the partials in one order.
// `turn` alternates between a block's rows: a warp may write its next partial while others still read the last ones.
template <bool kTop>
__device__ __forceinline__ Stats reduce_row(Stats s, int group, int turn = 0) {
    const int width = group < 32 ? group : 32;
    for (int d = width >> 1; d > 0; d >>= 1) {
        s.sum += __shfl_xor_sync(0xffffffffu, s.sum, d);
        if (kTop) s.top = max_nan(s.top, __shfl_xor_sync(0xffffffffu, s.top, d));
    }
    if (group > 32) {
        __shared__ Stats part[2][32];
        if ((threadIdx.x & 31) == 0) part[turn][threadIdx.x >> 5] = s;
        __syncthreads();
        const int first = (threadIdx.x & ~(group - 1)) >> 5;
        s = part[turn][first];
        for (int i = 1; i < (group >> 5); ++i) {
            s.sum += part[turn][first + i].sum;
            if (kTop) s.top = max_nan(s.top, part[turn][first + i].top);
        }
    }
    return s;
}

// 32 bytes at once: two 16-byte stores per lane would each write every other half of the sectors.
__device__ __forceinline__ void store_global32(float* p, const float (&v)[8]) {
    asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]),
                 "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7])
                 : "memory");
}

// What turns v * w into the stored value, from the row's statistics: v * w * first * second.
struct Factors {
    float first, second;
};

// For e4m3 the two factors are rstd and 1 / scale.  Each is finite (eps > 0, scale >= 2^-126), but their product, 448 / max|v w|
// unless the scale is at its lower bound, overflows for rows of values below 1.4e-36: only there the values take them one after the
// other, everywhere else their product alone.
__device__ __forceinline__ Factors row_factors(const NormParams& p, const Stats& s, float& scale) {
    const float rstd = p.norm ? rsqrtf(s.sum * p.inv_dim + p.eps) : 1.0f;
    if (!p.scales) return {1.0f, rstd};
    const float top = s.top * rstd;
    scale = top == 0.0f ? 1.0f : max_nan(top / kE4m3Max, kMinScale);
    const float inverse = 1.0f / scale, both = rstd * inverse;
    return both > kMaxFloat ? Factors{rstd, inverse} : Factors{1.0f, both};
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

// Few rows that start on 16-byte boundaries: one row per `group` threads, kV runs of 16 bytes per thread.
template <typename T, int kE, int kV>
__global__ void __launch_bounds__(1024) norm_row_kernel(const NormParams p) {
    allow_next_kernel();
    wait_for_kernels_before();
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
    s = reduce_row<true>(s, p.group);
    float scale = 1.0f;
    const Factors f = row_factors(p, s, scale);
    if (!live) return;
    if (p.scales && lane == 0) p.scales[row] = scale;
#pragma unroll
    for (int j = 0; j < kV; ++j) {
        const int at = (lane + j * p.group) * kE;
        if (at >= p.dim) continue;
        if (f.first != 1.0f)
#pragma unroll
            for (int i = 0; i < kE; ++i) v[j][i] *= f.first;
#pragma unroll
        for (int i = 0; i < kE; ++i) v[j][i] *= f.second;
        store_run<T, kE>(p, row * p.dim + at, v[j]);
    }
}

// Many rows: the same row per `group` threads, by blocks that stay and walk the rows.  Every thread copies its own runs
// of the row after next into shared memory (cp.async, 16 bytes each) while it works on the present one, and reads
// back only what it copied itself, so the copies need no barrier.  What bounds a norm is the bytes in flight:
// norm_row_kernel has them only between a block's start and its reduction (75600 x 5120 bf16 with a residual: 581 us
// = 5.3 TB/s; this one 471 us = 6.6 TB/s).  Two rows ahead; with three or four, fewer blocks fit (516, 592 us).
__device__ __forceinline__ void copy_async16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
// The same through L1, for two copies that share a sector: it comes from L2 once (75600 x 5120 bf16 with an fp32 residual
// 931 us past L1, 780 through it, 5.95 TB/s).
__device__ __forceinline__ void copy_async16_shared_sector(uint32_t to, const void* from) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}

constexpr int kAhead = 2;  // rows in flight per group

// kE elements as packed pairs of fp32.  Two of the values' steps then take one instruction: at 16 instructions per
// element (single values) the quantised form without a residual issued in 68 % of all cycles (75600 x 5120 bf16:
// 279 us; 262 with pairs, 238 with 80 registers a thread and so more blocks).
template <typename T, int kE>
struct Pairs {
    uint64_t p[kE / 2];
    __device__ __forceinline__ void from16(const uint4& raw) {  // 16 bytes of T
        const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
        if constexpr (sizeof(T) == 4) {
            p[0] = pack2(__uint_as_float(w[0]), __uint_as_float(w[1]));
            p[1] = pack2(__uint_as_float(w[2]), __uint_as_float(w[3]));
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (std::is_same_v<T, __half>) {
                    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
                    p[i] = pack2(f.x, f.y);
                } else {
                    p[i] = pack2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
                }
            }
        }
    }
    __device__ __forceinline__ void from_f32(const uint4& lo, const uint4& hi) {  // kE fp32 values (kE = 8)
        p[0] = pack2(__uint_as_float(lo.x), __uint_as_float(lo.y));
        p[1] = pack2(__uint_as_float(lo.z), __uint_as_float(lo.w));
        p[2 % (kE / 2)] = pack2(__uint_as_float(hi.x), __uint_as_float(hi.y));
        p[3 % (kE / 2)] = pack2(__uint_as_float(hi.z), __uint_as_float(hi.w));
    }
    __device__ __forceinline__ uint4 to16() const {
        uint32_t w[4];
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float lo, hi;
                unpack2(p[i], lo, hi);
                w[2 * i] = __float_as_uint(lo);
                w[2 * i + 1] = __float_as_uint(hi);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float lo, hi;
                unpack2(p[i], lo, hi);
                if constexpr (std::is_same_v<T, __half>) {
                    const __half2 h = __floats2half2_rn(lo, hi);
                    w[i] = *reinterpret_cast<const uint32_t*>(&h);
                } else {
                    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
                    w[i] = *reinterpret_cast<const uint32_t*>(&h);
                }
            }
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
};

// max(|a|, |b|, |c|), a NaN if any of them is one.
__device__ __forceinline__ float max_abs3(float a, float b, float c) {
    float d;
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// kRes: bytes of a residual run (0: no residual).
template <typename T, int kE, int kV, int kRes, bool kQuant>
__global__ void __launch_bounds__(kRes > 0 ? 512 : 768) norm_stream_kernel(const NormParams p) {
    extern __shared__ __align__(16) char smem[];
    constexpr int kPieces = 1 + kRes / 16;  // of 16 bytes: a thread's run of x, then of the residual
    const int lane = threadIdx.x & (p.group - 1);
    const int per_block = blockDim.x / p.group;
    const int64_t step = static_cast<int64_t>(gridDim.x) * per_block;
    const int64_t first = static_cast<int64_t>(blockIdx.x) * per_block + threadIdx.x / p.group;
    // The runs of this thread that exist are the first `runs`; the others stay zero in shared memory.
    const int runs = max(0, min(kV, ((p.dim + kE - 1) / kE - lane + p.group - 1) / p.group));
    const int hop = p.group * kE;  // elements from one run of a thread to its next
    const uint32_t base = static_cast<uint32_t>(__cvta_generic_to_shared(smem)) + threadIdx.x * 16;
    const uint32_t plane = blockDim.x * 16;  // the pieces of one instruction lie side by side
    auto place = [&](int slot, int j, int piece) { return base + ((slot * kV + j) * kPieces + piece) * plane; };
    // Short rows (kKeep): the weights stay in registers and the addresses move from row to row by a constant, 3 % of
    // the time of 393120 x 128; longer ones lose more by the registers (75600 x 5120 bf16 490 us instead of 472).
    constexpr bool kKeep = kV <= 2;
    constexpr int kResElem = kRes > 0 ? kRes / kE : 1;
    const T* const x = static_cast<const T*>(p.x) + lane * kE;
    const char* const res = static_cast<const char*>(p.residual) + lane * kRes;
    const T* x_next = x + first * p.x_stride;
    const char* res_next = res + first * p.residual_stride * kResElem;
    const int64_t x_step = step * p.x_stride, res_step = step * p.residual_stride * kResElem;
    auto fetch = [&](int64_t row, int slot) {
        if (row < p.rows) {
            const T* xr = kKeep ? x_next : x + row * p.x_stride;
            const char* rr = kKeep ? res_next : res + row * p.residual_stride * kResElem;
#pragma unroll
            for (int j = 0; j < kV; ++j) {
                if (j >= runs) break;
                copy_async16(place(slot, j, 0), xr + j * hop);
#pragma unroll
                for (int q = 0; q < kRes / 16; ++q) {
                    if constexpr (kRes == 32) copy_async16_shared_sector(place(slot, j, 1 + q), rr + j * hop * kResElem + q * 16);
                    else copy_async16(place(slot, j, 1 + q), rr + j * hop * kResElem + q * 16);
                }
            }
        }
        x_next += x_step;
        res_next += res_step;
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    auto weight_run = [&](int j) {
        Pairs<T, kE> w;
        const int at = lane * kE + j * hop;
        if (!p.weight_fp32) {
            w.from16(__ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(p.weight) + at)));
        } else {
            const uint4* q = reinterpret_cast<const uint4*>(static_cast<const float*>(p.weight) + at);
            if constexpr (kE == 8) w.from_f32(__ldg(q), __ldg(q + 1));
            else w.from16(__ldg(q));
        }
        return w;
    };
    for (int slot = 0; slot < kAhead; ++slot)
        for (int j = runs; j < kV; ++j)
            for (int q = 0; q < kPieces; ++q) store_shared16(place(slot, j, q), make_uint4(0, 0, 0, 0));
    allow_next_kernel();
    wait_for_kernels_before();
    for (int i = 0; i < kAhead; ++i) fetch(first + i * step, i);
    Pairs<T, kE> kept[kKeep ? kV : 1];
    if (kKeep && p.weight)
#pragma unroll
        for (int j = 0; j < kV; ++j)
            if (j < runs) kept[j % (kKeep ? kV : 1)] = weight_run(j);
    int64_t o_next = first * p.dim + lane * kE;
    const int64_t o_step = step * p.dim;
    int slot = 0, turn = 0;
    // Every thread of the block makes the same number of rounds: the reduction of wide groups is a block barrier.
    for (int64_t row = first; row - threadIdx.x / p.group < p.rows; row += step, o_next += o_step) {
        const bool live = row < p.rows;
        const int64_t o = kKeep ? o_next : row * p.dim + lane * kE;
        asm volatile("cp.async.wait_group %0;" ::"n"(kAhead - 1) : "memory");
        Pairs<T, kE> v[kV];
#pragma unroll
        for (int j = 0; j < kV; ++j) {
            v[j].from16(load_shared16(place(slot, j, 0)));
            if constexpr (kRes > 0) {
                Pairs<T, kE> r;
                if constexpr (kRes == 32) r.from_f32(load_shared16(place(slot, j, 1)), load_shared16(place(slot, j, 2)));
                else r.from16(load_shared16(place(slot, j, 1)));
#pragma unroll
                for (int i = 0; i < kE / 2; ++i) v[j].p[i] = add2(v[j].p[i], r.p[i]);
            }
        }
        fetch(row + kAhead * step, slot);
        if (++slot == kAhead) slot = 0;
        uint64_t sum2 = 0;
        float top = 0.0f;
#pragma unroll
        for (int j = 0; j < kV; ++j) {
            if constexpr (kRes == 32) {
                if (live && j < runs) {
                    float* at = static_cast<float*>(p.residual_out) + o + j * hop;
                    float f[8];
#pragma unroll
                    for (int i = 0; i < 4; ++i) unpack2(v[j].p[i % (kE / 2)], f[2 * i], f[2 * i + 1]);
                    if (p.residual_out32) {
                        store_global32(at, f);
                    } else {
                        *reinterpret_cast<float4*>(at) = make_float4(f[0], f[1], f[2], f[3]);
                        *reinterpret_cast<float4*>(at + 4) = make_float4(f[4], f[5], f[6], f[7]);
                    }
                }
            } else if constexpr (kRes > 0) {
                if (live && j < runs) *reinterpret_cast<uint4*>(static_cast<T*>(p.residual_out) + o + j * hop) = v[j].to16();
            }
#pragma unroll
            for (int i = 0; i < kE / 2; ++i) sum2 = fma2(v[j].p[i], v[j].p[i], sum2);
            if (p.weight && j < runs) {
                const Pairs<T, kE> w = kKeep ? kept[j % (kKeep ? kV : 1)] : weight_run(j);
#pragma unroll
                for (int i = 0; i < kE / 2; ++i) v[j].p[i] = mul2(v[j].p[i], w.p[i]);
            }
            if constexpr (kQuant) {
#pragma unroll
                for (int i = 0; i < kE / 2; ++i) {
                    float lo, hi;
                    unpack2(v[j].p[i], lo, hi);
                    top = max_abs3(top, lo, hi);
                }
            }
        }
        Stats s;
        {
            float lo, hi;
            unpack2(sum2, lo, hi);
            s = {lo + hi, top};
        }
        s = reduce_row<kQuant>(s, p.group, turn);
        turn ^= 1;
        float scale = 1.0f;
        const Factors f = row_factors(p, s, scale);
        if (!live) continue;
        if (kQuant && lane == 0) p.scales[row] = scale;
        if (kQuant && f.first != 1.0f) {
            const uint64_t f1 = pack2(f.first, f.first);
#pragma unroll
            for (int j = 0; j < kV; ++j)
#pragma unroll
                for (int i = 0; i < kE / 2; ++i) v[j].p[i] = mul2(v[j].p[i], f1);
        }
        const uint64_t f2 = pack2(f.second, f.second);
#pragma unroll
        for (int j = 0; j < kV; ++j) {
            if (j >= runs) break;
#pragma unroll
            for (int i = 0; i < kE / 2; ++i) v[j].p[i] = mul2(v[j].p[i], f2);
            if constexpr (kQuant) {
                uint16_t h[4];
#pragma unroll
                for (int i = 0; i < kE / 2; ++i) {
                    float lo, hi;
                    unpack2(v[j].p[i], lo, hi);
                    h[i] = e4m3x2(lo, hi);
                }
                uint8_t* at = static_cast<uint8_t*>(p.out) + o + j * hop;
                const uint32_t lo = h[0] | (static_cast<uint32_t>(h[1]) << 16);
                if constexpr (kE == 8) *reinterpret_cast<uint2*>(at) = make_uint2(lo, h[2] | (static_cast<uint32_t>(h[3]) << 16));
                else *reinterpret_cast<uint32_t*>(at) = lo;
            } else {
                *reinterpret_cast<uint4*>(static_cast<T*>(p.out) + o + j * hop) = v[j].to16();
            }
        }
    }
}

// Rows that neither fit 16-byte runs nor lie side by side: runs of four elements or single ones, straight from global memory, by blocks that
// stay.  A thread has the next row's runs on their way in registers while it works on the present row, and takes 16
// elements of it, because a row's reduction costs every thread the same whatever its share (20000 x 1001 bf16: a
// block of 256 threads per row, four elements each, issued 75 instructions per element and took 64 us).  kRes: 0 no residual, 1 in the type of x, 2 fp32.
template <typename T, int kE, int kV, int kRes>
__global__ void __launch_bounds__(512) norm_narrow_kernel(const NormParams p) {
    using R = std::conditional_t<kRes == 2, float, T>;
    const int lane = threadIdx.x & (p.group - 1);
    const int per_block = blockDim.x / p.group;
    const int64_t step = static_cast<int64_t>(gridDim.x) * per_block;
    const int64_t first = static_cast<int64_t>(blockIdx.x) * per_block + threadIdx.x / p.group;
    Run<T, kE> in[kV];
    Run<R, kE> add[kV];
    auto fetch = [&](int64_t row) {
        const T* x = static_cast<const T*>(p.x) + row * p.x_stride;
        const R* r = static_cast<const R*>(p.residual) + row * p.residual_stride;
#pragma unroll
        for (int j = 0; j < kV; ++j) {
            const int at = (lane + j * p.group) * kE;
            if (row >= p.rows || at >= p.dim) continue;
            in[j].load(x + at);
            if constexpr (kRes > 0) add[j].load(r + at);
        }
    };
    allow_next_kernel();
    wait_for_kernels_before();
    fetch(first);
    float w[kV][kE];  // a load of them within the loop would have to wait for the next row's runs as well
#pragma unroll
    for (int j = 0; j < kV; ++j) {
        const int at = (lane + j * p.group) * kE;
        if (at < p.dim) weights_of<T, kE>(p, at, w[j]);
    }
    int turn = 0;
    for (int64_t row = first; row - threadIdx.x / p.group < p.rows; row += step) {
        const bool live = row < p.rows;
        float v[kV][kE];
#pragma unroll
        for (int j = 0; j < kV; ++j)
#pragma unroll
            for (int i = 0; i < kE; ++i) v[j][i] = kRes > 0 ? in[j].get(i) + add[j].get(i) : in[j].get(i);
        fetch(row + step);
        Stats s = {0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < kV; ++j) {
            const int at = (lane + j * p.group) * kE;
            if (!live || at >= p.dim) continue;
            if constexpr (kRes > 0) {
                Run<R, kE> r;
#pragma unroll
                for (int i = 0; i < kE; ++i) r.set(i, v[j][i]);
                r.store(static_cast<R*>(p.residual_out) + row * p.dim + at);
            }
#pragma unroll
            for (int i = 0; i < kE; ++i) {
                s.sum += v[j][i] * v[j][i];
                v[j][i] *= w[j][i];
                if (p.scales) s.top = max_nan(s.top, fabsf(v[j][i]));
            }
        }
        s = p.scales ? reduce_row<true>(s, p.group, turn) : reduce_row<false>(s, p.group, turn);
        turn ^= 1;
        float scale = 1.0f;
        const Factors f = row_factors(p, s, scale);
        if (!live) continue;
        if (p.scales && lane == 0) p.scales[row] = scale;
#pragma unroll
        for (int j = 0; j < kV; ++j) {
            const int at = (lane + j * p.group) * kE;
            if (at >= p.dim) continue;
            if (f.first != 1.0f)
#pragma unroll
                for (int i = 0; i < kE; ++i) v[j][i] *= f.first;
#pragma unroll
            for (int i = 0; i < kE; ++i) v[j][i] *= f.second;
            store_run<T, kE>(p, row * p.dim + at, v[j]);
        }
    }
}

// Stores elements [lo, hi) of a run, given as pairs of elements; at least one end is the run's own.
template <typename P, int kPairs>
__device__ __forceinline__ void store_part(P* at, const P (&v)[kPairs], int lo, int hi) {
    using Half = std::conditional_t<sizeof(P) == 8, uint32_t, std::conditional_t<sizeof(P) == 4, uint16_t, uint8_t>>;
    using Two = typename Raw<2 * sizeof(P)>::type;
    constexpr int kE = 2 * kPairs;
    union Twos {
        P p[2];
        Two two;
        __device__ __forceinline__ Twos() {}
    } t;
    if (lo == 0 && hi == kE) {
        if constexpr (kPairs * sizeof(P) <= 16) {
            union {
                P p[kPairs];
                typename Raw<kPairs * sizeof(P)>::type all;
            } u;
#pragma unroll
            for (int i = 0; i < kPairs; ++i) u.p[i] = v[i];
            *reinterpret_cast<decltype(u.all)*>(at) = u.all;
        } else {
#pragma unroll
            for (int i = 0; i < kPairs; i += 2) {
                t.p[0] = v[i];
                t.p[1] = v[i + 1];
                *reinterpret_cast<Two*>(at + i) = t.two;
            }
        }
        return;
    }
    // A part of `count` elements is four, two and one of them, each on an address that its size divides.
    const bool front = lo == 0;
    const int count = front ? hi : kE - lo;
    auto pick = [&](int q) {
        P r = v[0];
#pragma unroll
        for (int i = 1; i < kPairs; ++i)
            if (q == i) r = v[i];
        return r;
    };
    if constexpr (kPairs == 4) {
        if (count & 4) {
            t.p[0] = front ? v[0] : v[2];
            t.p[1] = front ? v[1] : v[3];
            *reinterpret_cast<Two*>(at + (front ? 0 : 2)) = t.two;
        }
    }
    if (count & 2) {
        const int q = front ? (count & 4) / 2 : kPairs - 1 - (count & 4) / 2;
        at[q] = pick(q);
    }
    if (count & 1) {
        const int q = front ? count >> 1 : kPairs - 1 - (count >> 1);
        const P pair = pick(q);
        reinterpret_cast<Half*>(at)[2 * q + (front ? 0 : 1)] = static_cast<Half>(front ? pair : pair >> (4 * sizeof(P)));
    }
}

template <typename T>
__device__ __forceinline__ auto pair_of(float lo, float hi) {
    if constexpr (sizeof(T) == 4) return pack2(lo, hi);
    else if constexpr (std::is_same_v<T, __half>) {
        const __half2 h = __floats2half2_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&h);
    } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
}

// Contiguous rows of a width that 16-byte runs do not divide.  The runs are those of the whole array, so a row starts
// somewhere within its first one, and a run that two rows share is read by both and written in parts.  The weights, whose
// place in a run differs from row to row, lie in shared memory as fp32, with a gap after every 32 for its banks.
// Bound by instruction issue (bf16 with a residual 20000 x 1001 40 us, single elements 82, HBM 25; 6000 x 5121 54, 124, 38).
__device__ __forceinline__ int banked(int i) { return i + (i >> 5); }

template <int kE, typename W>
__device__ __forceinline__ void stage_weights(float* to, const W* w, int dim) {
    constexpr int kBatch = 8;  // loads on their way at once (one by one 5121 weights took 7 us)
    for (int i0 = threadIdx.x; i0 < dim + 2 * kE; i0 += blockDim.x * kBatch) {
        float v[kBatch];
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
            const int i = i0 + b * blockDim.x - kE;
            v[b] = i >= 0 && i < dim ? to_f32(w[i]) : 0.0f;
        }
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
            const int i = i0 + b * blockDim.x;
            if (i < dim + 2 * kE) to[banked(i)] = v[b];
        }
    }
}

template <typename T, int kV, int kRes>
__global__ void __launch_bounds__(512) norm_shifted_kernel(const NormParams p) {
    using R = std::conditional_t<kRes == 2, float, T>;
    constexpr int kE = 16 / sizeof(T);
    extern __shared__ float weights[];  // [kE zeros | dim | kE zeros]
    const int lane = threadIdx.x & (p.group - 1);
    const int per_block = blockDim.x / p.group;
    const int64_t step = static_cast<int64_t>(gridDim.x) * per_block;
    const int64_t first = static_cast<int64_t>(blockIdx.x) * per_block + threadIdx.x / p.group;
    const int64_t total = p.rows * p.dim;
    const T* const x = static_cast<const T*>(p.x);
    const R* const residual = static_cast<const R*>(p.residual);
    auto shift_of = [&](int64_t row) { return (static_cast<int>(row) & (kE - 1)) * (p.dim & (kE - 1)) & (kE - 1); };
    Run<T, kE> in[kV];
    Run<R, kE> add[kV];
    auto fetch = [&](int64_t row) {
        if (row >= p.rows) return;
        const int shift = shift_of(row);
        const int64_t start = row * p.dim - shift;
#pragma unroll
        for (int j = 0; j < kV; ++j) {
            const int c = (lane + j * p.group) * kE;
            if (c - shift >= p.dim) continue;
            if (start + c + kE <= total) {
                in[j].load(x + start + c);
                if constexpr (kRes > 0) add[j].load(residual + start + c);
            } else {  // the array ends within this run
#pragma unroll
                for (int i = 0; i < kE; ++i)
                    if (start + c + i < total) {
                        in[j].d.elem[i] = x[start + c + i];
                        if constexpr (kRes > 0) add[j].d.elem[i] = residual[start + c + i];
                    }
            }
        }
    };
    allow_next_kernel();
    wait_for_kernels_before();
    fetch(first);
    if (p.weight) {
        if (p.weight_fp32) stage_weights<kE>(weights, static_cast<const float*>(p.weight), p.dim);
        else stage_weights<kE>(weights, static_cast<const T*>(p.weight), p.dim);
        __syncthreads();
    }
    int turn = 0;
    for (int64_t row = first; row - threadIdx.x / p.group < p.rows; row += step) {
        const bool live = row < p.rows;
        const int shift = shift_of(row);
        const int64_t start = row * p.dim - shift;
        float v[kV][kE];
#pragma unroll
        for (int j = 0; j < kV; ++j) {
#pragma unroll
            for (int i = 0; i < kE; ++i) v[j][i] = kRes > 0 ? in[j].get(i) + add[j].get(i) : in[j].get(i);
            const int at = (lane + j * p.group) * kE - shift;
            if (at < 0 || at + kE > p.dim)
#pragma unroll
                for (int i = 0; i < kE; ++i)
                    if (at + i < 0 || at + i >= p.dim) v[j][i] = 0.0f;
        }
        fetch(row + step);
        Stats s = {0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < kV; ++j) {
            const int at = (lane + j * p.group) * kE - shift;
            if (!live || at >= p.dim) continue;
            if constexpr (kRes > 0) {
                decltype(pair_of<R>(0.0f, 0.0f)) pairs[kE / 2];
#pragma unroll
                for (int i = 0; i < kE / 2; ++i) pairs[i] = pair_of<R>(v[j][2 * i], v[j][2 * i + 1]);
                store_part(reinterpret_cast<decltype(&pairs[0])>(static_cast<R*>(p.residual_out) + start + shift + at), pairs,
                           max(0, -at), min(kE, p.dim - at));
            }
#pragma unroll
            for (int i = 0; i < kE; ++i) {
                s.sum += v[j][i] * v[j][i];
                if (p.weight) v[j][i] *= weights[banked(at + kE + i)];
                if (p.scales) s.top = max_nan(s.top, fabsf(v[j][i]));
            }
        }
        s = p.scales ? reduce_row<true>(s, p.group, turn) : reduce_row<false>(s, p.group, turn);
        turn ^= 1;
        float scale = 1.0f;
        const Factors f = row_factors(p, s, scale);
        if (!live) continue;
        if (p.scales && lane == 0) p.scales[row] = scale;
        if (f.first != 1.0f)
#pragma unroll
            for (int j = 0; j < kV; ++j)
#pragma unroll
                for (int i = 0; i < kE; ++i) v[j][i] *= f.first;
#pragma unroll
        for (int j = 0; j < kV; ++j) {
            const int at = (lane + j * p.group) * kE - shift;
            if (at >= p.dim) continue;
            const int lo = max(0, -at), hi = min(kE, p.dim - at);
            if (p.scales) {
                uint16_t pairs[kE / 2];
#pragma unroll
                for (int i = 0; i < kE / 2; ++i) pairs[i] = e4m3x2(v[j][2 * i] * f.second, v[j][2 * i + 1] * f.second);
                store_part(reinterpret_cast<uint16_t*>(static_cast<uint8_t*>(p.out) + start + shift + at), pairs, lo, hi);
            } else {
                decltype(pair_of<T>(0.0f, 0.0f)) pairs[kE / 2];
#pragma unroll
                for (int i = 0; i < kE / 2; ++i) pairs[i] = pair_of<T>(v[j][2 * i] * f.second, v[j][2 * i + 1] * f.second);
                store_part(reinterpret_cast<decltype(&pairs[0])>(static_cast<T*>(p.out) + start + shift + at), pairs, lo, hi);
            }
        }
    }
}

// Rows too long for the registers of a block: one block per row, the row read twice (the second time from L2).
template <typename T>
__global__ void __launch_bounds__(1024) norm_long_kernel(const NormParams p) {
    allow_next_kernel();
    wait_for_kernels_before();
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
    s = reduce_row<true>(s, p.group);
    float scale = 1.0f;
    const Factors f = row_factors(p, s, scale);
    if (p.scales && threadIdx.x == 0) p.scales[row] = scale;
    for (int at = threadIdx.x; at < p.dim; at += blockDim.x) {
        const float y[1] = {value(at) * weight(at) * f.first * f.second};
        store_run<T, 1>(p, row * p.dim + at, y);
    }
}

constexpr int kSms = 148;
constexpr int kStreamBlocks = 4 * kSms;

constexpr int kMaxSmem = 226 * 1024;  // of 227 KB, beside the partials of the reduction

// A launch whose start may overlap the end of the kernel before it (each kernel waits before its first access to memory).
cudaError_t launch(void (*kernel)(NormParams), const NormParams& p, int64_t blocks, int threads, int smem, cudaStream_t stream) {
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(blocks));
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, p);
}

template <int kV, int kRes>
constexpr int stream_smem(int threads) { return kAhead * kV * (16 + kRes) * threads; }

template <typename T, int kE, int kV, int kRes, bool kQuant>
cudaError_t launch_stream_as(const NormParams& p, int threads, cudaStream_t stream) {
    auto kernel = norm_stream_kernel<T, kE, kV, kRes, kQuant>;
    const int smem = stream_smem<kV, kRes>(threads);
    // Resident blocks per SM, asked once for each block size (128, 256 or 512 threads) and device.
    constexpr int kMaxDevices = 64;
    static std::atomic<int> resident[kMaxDevices][3];
    int dev = 0;
    cudaError_t err = cudaGetDevice(&dev);
    if (err != cudaSuccess) return err;
    std::atomic<int>& known = resident[dev % kMaxDevices][threads / 256];
    int per_sm = known.load(std::memory_order_acquire);
    if (per_sm == 0) {
        err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem);
        if (err == cudaSuccess) err = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, threads, smem);
        if (err != cudaSuccess) return err;
        per_sm = std::max(per_sm, 1);
        known.store(per_sm, std::memory_order_release);
    }
    const int64_t blocks = (p.rows + threads / p.group - 1) / (threads / p.group);
    return launch(kernel, p, std::min<int64_t>(blocks, static_cast<int64_t>(kSms) * per_sm), threads, smem, stream);
}

template <typename T, int kE, int kV, int kRes>
cudaError_t launch_stream(const NormParams& p, int threads, cudaStream_t stream) {
    return p.scales ? launch_stream_as<T, kE, kV, kRes, true>(p, threads, stream)
                    : launch_stream_as<T, kE, kV, kRes, false>(p, threads, stream);
}

constexpr int kMostRuns = 6, kMostWithResidual = 3;  // of 16 bytes, by one thread of a block of up to 512 (launch_rows)
static_assert(stream_smem<kMostRuns, 0>(512) <= kMaxSmem && stream_smem<kMostWithResidual, 32>(512) <= kMaxSmem, "shared memory of the stream kernel");

// Rows of 16-byte runs.
template <typename T, int kV>
cudaError_t launch_wide(const NormParams& p, int threads, cudaStream_t stream) {
    constexpr int kE = 16 / sizeof(T);
    const int64_t blocks = (p.rows + threads / p.group - 1) / (threads / p.group);
    // Worth its longer start only where a block walks several rows: 2000 rows of 5120 bf16 with a residual 15.6 us
    // (norm_row_kernel 17.4), 300 rows as fast either way.
    if (blocks > kStreamBlocks && threads <= 512) {
        if (!p.residual) return launch_stream<T, kE, kV, 0>(p, threads, stream);
        if constexpr (kV <= kMostWithResidual) {  // more runs come with blocks of 1024 threads alone (launch_rows)
            if (p.residual_fp32) return launch_stream<T, kE, kV, 4 * kE>(p, threads, stream);
            return launch_stream<T, kE, kV, 16>(p, threads, stream);
        }
    }
    return launch(norm_row_kernel<T, kE, kV>, p, blocks, threads, 0, stream);
}

template <typename T, int kE, int kV>
cudaError_t launch_narrow(const NormParams& p, int threads, cudaStream_t stream) {
    const int64_t blocks = (p.rows + threads / p.group - 1) / (threads / p.group);
    const int64_t grid = std::min<int64_t>(blocks, kSms * (1024 / threads));
    if (!p.residual) return launch(norm_narrow_kernel<T, kE, kV, 0>, p, grid, threads, 0, stream);
    if (!p.residual_fp32) return launch(norm_narrow_kernel<T, kE, kV, 1>, p, grid, threads, 0, stream);
    return launch(norm_narrow_kernel<T, kE, kV, 2>, p, grid, threads, 0, stream);
}

template <typename T, int kV>
cudaError_t launch_shifted(const NormParams& p, int threads, int smem, cudaStream_t stream) {
    const int64_t blocks = (p.rows + threads / p.group - 1) / (threads / p.group);
    const int64_t grid = std::min<int64_t>(blocks, kSms * (1024 / threads));
    if (!p.residual) return launch(norm_shifted_kernel<T, kV, 0>, p, grid, threads, smem, stream);
    if (!p.residual_fp32) return launch(norm_shifted_kernel<T, kV, 1>, p, grid, threads, smem, stream);
    return launch(norm_shifted_kernel<T, kV, 2>, p, grid, threads, smem, stream);
}

constexpr int kShiftedMost = 3;         // runs of a thread
constexpr int kShiftedMaxDim = 11000;   // the weights in 48 KB of shared memory

constexpr int kHalfRunsMaxDim = 512 * 16;  // 16 elements per thread of the largest block of norm_narrow_kernel

template <typename T>
cudaError_t launch_shifted(NormParams p, cudaStream_t stream) {
    constexpr int kE = 16 / sizeof(T);
    const int runs = (p.dim + 2 * kE - 2) / kE;  // of a row that starts on the last element of one
    p.group = 1;
    while (p.group < 512 && p.group * kShiftedMost < runs) p.group *= 2;
    const int threads = std::max(p.group, 128), smem = p.weight ? (p.dim + 2 * kE) / 32 * 132 + 132 : 0;
    switch ((runs + p.group - 1) / p.group) {
        case 1: return launch_shifted<T, 1>(p, threads, smem, stream);
        case 2: return launch_shifted<T, 2>(p, threads, smem, stream);
        default: return launch_shifted<T, kShiftedMost>(p, threads, smem, stream);
    }
}

template <typename T, int kE>
cudaError_t launch_rows(NormParams p, cudaStream_t stream) {
    const int runs = (p.dim + kE - 1) / kE;
    constexpr bool kWide = kE * sizeof(T) == 16;
    // The smallest group of threads that holds the row in so many runs each: three 16-byte runs (75600 x 5120 bf16
    // with a residual 471 us, with six runs 490), six where the rows are wide, have no residual and are many enough for
    // norm_stream_kernel (quantised 238 us, three 311: the reduction over twice the warps costs more than the loads).
    // Fewer rows of that kind take three: bf16 300 x 5120 3.5 us, six 5.2; 590 x 6144 4.0 and 9.4 (registers of
    // norm_row_kernel spill); from 592 rows on it is about even (1000 x 5120 5.5 and 5.6, quantised 5.9 and 5.7).
    const int most = !kWide ? 16 / kE : p.residual || runs <= 384 || p.rows <= kStreamBlocks ? kMostWithResidual : kMostRuns;
    int group = 1;
    while (group < 512 && group * most < runs) group *= 2;
    int per_thread = (runs + group - 1) / group;
    if (kWide && per_thread > most) {
        group = 1024;
        per_thread = (runs + group - 1) / group;
    }
    if (per_thread > (kWide ? kMostRuns : most)) {
        p.group = 1024;
        return launch(norm_long_kernel<T>, p, p.rows, 1024, 0, stream);
    }
    p.group = group;
    const int threads = group > 128 ? group : 128;
    if constexpr (kWide) {
        switch (per_thread) {
            case 1: return launch_wide<T, 1>(p, threads, stream);
            case 2: return launch_wide<T, 2>(p, threads, stream);
            case 3: return launch_wide<T, 3>(p, threads, stream);
            case 4: return launch_wide<T, 4>(p, threads, stream);
            case 5: return launch_wide<T, 5>(p, threads, stream);
            default: return launch_wide<T, 6>(p, threads, stream);
        }
    } else if constexpr (kE == 4) {
        if (per_thread <= 2) return launch_narrow<T, 4, 2>(p, threads, stream);
        return launch_narrow<T, 4, 4>(p, threads, stream);
    } else {
        if (per_thread <= 4) return launch_narrow<T, 1, 4>(p, threads, stream);
        if (per_thread <= 8) return launch_narrow<T, 1, 8>(p, threads, stream);
        if (per_thread <= 12) return launch_narrow<T, 1, 12>(p, threads, stream);
        return launch_narrow<T, 1, 16>(p, threads, stream);
    }
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
    constexpr int kWide = 16 / sizeof(T);
    if (fits(kWide)) return launch_rows<T, kWide>(p, stream);
    auto starts = [](const void* base, int bytes) { return reinterpret_cast<uintptr_t>(base) % bytes == 0; };
    const bool packed = (p.rows == 1 || (p.x_stride == p.dim && (!p.residual || p.residual_stride == p.dim))) && starts(p.x, 16) &&
                        starts(p.residual, 16) && starts(p.residual_out, 16) && starts(p.out, p.scales ? kWide : 16);
    // Runs of half the width suit rows that they divide, as long as no residual adds to the loads or the rows are short
    // (bf16, half / shared whole ones: 20000 x 1004 20 / 27 us, with a residual 34 / 40; 10000 x 1500 19 / 22 and 31 / 28;
    // 6000 x 5124 42 / 44 and 66 / 53), and as long as a block's registers hold the row (6000 x 8196 shared 87, and 186 by
    // norm_long_kernel).
    if constexpr (kWide == 8) {
        if (fits(4) && ((!p.residual && p.dim <= kHalfRunsMaxDim) || p.dim <= 1024 || !packed)) return launch_rows<T, 4>(p, stream);
    }
    if (packed && p.dim >= kWide && p.dim <= kShiftedMaxDim && p.dim <= kWide * (512 * kShiftedMost - 2)) return launch_shifted<T>(p, stream);
    return launch_rows<T, 1>(p, stream);
}

}  // namespace
}  // namespace sdb

using namespace sdb;

extern "C" int mindiesd_add_rms_norm(const mindiesd_norm_args* a, void* stream_) {
    if (!a || !a->x || !a->out) return MINDIESD_E_NULL;
    if ((a->residual == nullptr) != (a->residual_out == nullptr)) return MINDIESD_E_NULL;
    if (a->rows <= 0 || a->dim <= 0) return MINDIESD_E_SHAPE;
    if (a->rows > 0x7fffffff || a->dim > 0x3fffffff) return MINDIESD_E_CAPACITY;  // blocks of a grid, 32-bit columns
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
    // Rows are fetched ahead, and long ones read twice, so nothing may be written where an input is still read, nor where
    // another output is written.
    struct Span {
        uintptr_t first, end;
        bool written;
    };
    auto span = [](const void* at, int64_t rows, int64_t stride, int64_t width, int bytes, bool written) {
        const uintptr_t first = reinterpret_cast<uintptr_t>(at);
        return Span{first, at ? first + static_cast<uintptr_t>((rows - 1) * stride + width) * bytes : first, written};
    };
    const int oe = dtype_bytes(a->out_dtype), re = a->residual ? dtype_bytes(a->residual_dtype) : 0;
    const Span spans[] = {span(a->x, a->rows, a->x_stride, a->dim, e, false),
                          span(a->residual, a->rows, a->residual_stride, a->dim, re, false),
                          span(a->weight, 1, 0, a->dim, a->weight ? dtype_bytes(a->weight_dtype) : 0, false),
                          span(a->out, a->rows, a->dim, a->dim, oe, true),
                          span(a->residual_out, a->rows, a->dim, a->dim, re, true),
                          span(a->out_dtype == MINDIESD_E4M3 ? a->scales : nullptr, a->rows, 1, 1, 4, true)};
    for (const Span& s : spans)
        for (const Span& t : spans)
            if (&s != &t && s.written && s.first < t.end && t.first < s.end) return MINDIESD_E_VALUE;
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
    p.residual_out32 = aligned(a->residual_out, 32) && static_cast<int64_t>(a->dim) * re % 32 == 0;
    p.norm = a->quant_only ? 0 : 1;
    p.eps = a->eps;
    p.inv_dim = 1.0f / static_cast<float>(a->dim);
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    cudaError_t err;
    if (a->dtype == MINDIESD_BF16) err = launch_typed<__nv_bfloat16>(p, stream);
    else if (a->dtype == MINDIESD_FP16) err = launch_typed<__half>(p, stream);
    else err = launch_typed<float>(p, stream);
    if (err == cudaSuccess) return MINDIESD_OK;
    cudaGetLastError();  // the caller gets the error from here; the next call's check must not find it again
    return static_cast<int>(err);
}
