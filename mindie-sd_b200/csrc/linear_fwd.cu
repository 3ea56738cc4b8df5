// Matrix product with its epilogue:  out = residual + gate * act(x w^T * scales + bias).
//   x [m, k], w [n, k] (both k-contiguous), bf16 / fp16 / e4m3 operands, fp32 accumulation, one rounding of the result.
//
// Two kernels.  Both stream 128-byte wide tiles of x and w through a ring of shared-memory stages filled by a TMA
// thread, and one thread issues tcgen05 MMAs into tensor memory.
//
// `linear_pair_kernel` (many rows): persistent, two thread blocks (a cluster on neighbouring SMs) work on one
// 256 x tile_n tile with two-SM MMAs, so each SM fetches 128 rows of x and only HALF of the tile's rows of w: 32 KB
// per 128 x 256 x 128-byte step.  Two accumulators of up to 256 columns: the epilogue of a tile (eight warps per block)
// runs under the MMAs of the next one.
//
// `linear_swap_kernel` (few rows): the time is that of reading w once, so w takes the M side of the MMA (128 of
// its rows per thread block) and the tokens, rounded up to 16, the N side.  Where n / 128 thread blocks would not
// fill the GPU, k is split over the blocks of a cluster; they leave their fp32 partials in shared memory and
// every block adds a share of the tokens in the order of the ranks over distributed shared memory: no workspace,
// no atomics, the same bits every time.
#include "capi_common.h"
#include "ptx_sm100.cuh"
#include "row_io.cuh"

namespace sdb {
namespace {

constexpr int kStepBytes = 128;             // bytes of k per ring stage (one swizzle row)
constexpr int kRowTile = 128 * kStepBytes;  // 16 KB: 128 rows of one stage
constexpr int kStatusLinearGaveUp = 105;

enum Act { kNone = 0, kRelu = 1, kSilu = 2, kGelu = 3, kGeluTanh = 4 };

struct Epilogue {
    const void* bias;
    const void* residual;  // in the output's type
    const void* gate;
    const float* x_scale;
    const float* w_scale;
    void* out;
    int64_t residual_stride, out_stride, gate_stride;
    uint32_t rows_per_gate;
    int x_scale_step, w_scale_step;  // 0: one scale for all
    int bias_type, gate_type;        // MINDIESD_BF16 / FP16 / FP32
    int out_fp16, act;
    int wide_out, wide_residual, wide_cols;  // rows (column vectors) can be moved 16 bytes at a time
    int m, n;
};

struct LinearParams {
    alignas(64) CUtensorMap tm_x;
    alignas(64) CUtensorMap tm_w;
    Epilogue e;
    int k_steps, k_step_elems;
    int tile_n;                    // pair kernel: columns of a tile; swap kernel: tokens of a tile
    int tiles_m, tiles_n, band;    // pair kernel: tiles are walked in bands of `band` row tiles
    int stages, tmem_cols, split;  // swap kernel
    uint32_t idesc;
    uint32_t wait_limit_us;
    int test_withhold;
    int* status;
};

__device__ __forceinline__ float load_any(const void* p, int type, int64_t i) {
    if (type == MINDIESD_FP32) return __ldg(static_cast<const float*>(p) + i);
    if (type == MINDIESD_BF16) return to_f32(static_cast<const __nv_bfloat16*>(p)[i]);
    return to_f32(static_cast<const __half*>(p)[i]);
}

__device__ __forceinline__ void unpack_pair(uint32_t w, int fp16, float& lo, float& hi) {
    if (fp16) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
        lo = f.x;
        hi = f.y;
    } else {
        lo = __uint_as_float(w << 16);
        hi = __uint_as_float(w & 0xffff0000u);
    }
}

__device__ __forceinline__ uint32_t pack_pair(float lo, float hi, int fp16) {
    if (fp16) {
        const __half2 h = __floats2half2_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    const __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&b);
}

// Eight consecutive column values (bias, gate, weight scale); every lane of a warp reads the same ones.
__device__ __forceinline__ void load_cols8(const void* p, int type, int64_t row_at, int col, int n, bool wide, float (&f)[8]) {
    if (wide && col + 8 <= n) {
        if (type == MINDIESD_FP32) {
            const float4* q = reinterpret_cast<const float4*>(static_cast<const float*>(p) + row_at + col);
            const float4 a = __ldg(q), b = __ldg(q + 1);
            f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
            f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
        } else {
            const uint4 a = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + row_at + col));
            unpack_pair(a.x, type == MINDIESD_FP16, f[0], f[1]);
            unpack_pair(a.y, type == MINDIESD_FP16, f[2], f[3]);
            unpack_pair(a.z, type == MINDIESD_FP16, f[4], f[5]);
            unpack_pair(a.w, type == MINDIESD_FP16, f[6], f[7]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = col + i < n ? load_any(p, type, row_at + col + i) : 0.0f;
    }
}

// The activations in the forms that keep their relative accuracy for large negative arguments:
//   gelu(v) = v/2 erfc(-v / sqrt 2),  silu(v) = v / (1 + e^-v),
//   gelu_tanh(v) = v/2 (1 + tanh u) = v / (1 + e^-2u),  u = sqrt(2/pi) (v + 0.044715 v^3).
__device__ __forceinline__ float silu(float v) { return __fdividef(v, 1.0f + __expf(-v)); }
__device__ __forceinline__ float gelu_tanh(float v) {
    const float u2 = v * fmaf(0.07135481627f, v * v, 1.595769122f);
    return __fdividef(v, 1.0f + __expf(-u2));
}
template <int kN>
__device__ __forceinline__ void activate(float (&v)[kN], int act) {
    switch (act) {
        case kRelu:
#pragma unroll
            for (int i = 0; i < kN; ++i) v[i] = v[i] < 0.0f ? 0.0f : v[i];  // a NaN stays
            break;
        case kSilu:
#pragma unroll
            for (int i = 0; i < kN; ++i) v[i] = silu(v[i]);
            break;
        case kGelu:
#pragma unroll
            for (int i = 0; i < kN; ++i) v[i] = 0.5f * v[i] * erfcf(-0.70710678118654752f * v[i]);
            break;
        case kGeluTanh:
#pragma unroll
            for (int i = 0; i < kN; ++i) v[i] = gelu_tanh(v[i]);
            break;
        default: break;
    }
}

__device__ __forceinline__ void report(const LinearParams& p, const volatile int* abort_flag) {
    if (*abort_flag && p.status && atomicCAS(p.status, 0, kStatusLinearGaveUp) == 0) {
        p.status[1] = abort_flag[1];
        p.status[2] = static_cast<int>(blockIdx.x);
        p.status[3] = static_cast<int>(blockIdx.y);
        p.status[4] = static_cast<int>(blockIdx.z);
    }
}

// ---- many rows ---------------------------------------------------------------------------------------------

constexpr int kPairThreads = 384;  // warps: 0 loader, 1 MMA, 2 tensor memory, 3 idle, 4..11 epilogue
constexpr int kPairStages = 6;
constexpr int kPairStageBytes = 2 * kRowTile;
constexpr int kStagingBytes = 32 * 64;  // per epilogue warp: 32 rows of 32 two-byte values
constexpr int kPairSmem = kPairStages * kPairStageBytes + 8 * kStagingBytes + 256 + 1024;

// Offset of 16-byte chunk c of row r in a warp's staging buffer; the exclusive or keeps both the row-wise writes and
// the chunk-wise reads free of bank conflicts.
__device__ __forceinline__ uint32_t staged(int r, int c) { return r * 64 + ((c ^ ((r >> 1) & 3)) << 4); }

// Moves the 32 x 32 block at (row0, col0) of a two-byte row-major matrix between global memory and the staging
// buffer; lanes cover 8 rows of 64 bytes at a time, or one row of 32 elements where 16-byte access is not possible.
__device__ __forceinline__ void stage_in(char* buf, const uint16_t* g, int64_t stride, int row0, int col0, int m, int n, bool wide,
                                         int lane) {
    if (wide) {
        const int c = lane & 3;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = i * 8 + (lane >> 2);
            uint4 v = make_uint4(0, 0, 0, 0);
            if (row0 + r < m && col0 + c * 8 < n)
                v = __ldg(reinterpret_cast<const uint4*>(g + static_cast<int64_t>(row0 + r) * stride + col0 + c * 8));
            *reinterpret_cast<uint4*>(buf + staged(r, c)) = v;
        }
    } else {
#pragma unroll 4
        for (int r = 0; r < 32; ++r) {
            uint16_t v = 0;
            if (row0 + r < m && col0 + lane < n) v = g[static_cast<int64_t>(row0 + r) * stride + col0 + lane];
            *reinterpret_cast<uint16_t*>(buf + staged(r, lane >> 3) + (lane & 7) * 2) = v;
        }
    }
}
__device__ __forceinline__ void stage_out(const char* buf, uint16_t* g, int64_t stride, int row0, int col0, int m, int n, bool wide,
                                          int lane) {
    if (wide) {
        const int c = lane & 3;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = i * 8 + (lane >> 2);
            if (row0 + r < m && col0 + c * 8 < n)
                *reinterpret_cast<uint4*>(g + static_cast<int64_t>(row0 + r) * stride + col0 + c * 8) =
                    *reinterpret_cast<const uint4*>(buf + staged(r, c));
        }
    } else {
#pragma unroll 4
        for (int r = 0; r < 32; ++r)
            if (row0 + r < m && col0 + lane < n)
                g[static_cast<int64_t>(row0 + r) * stride + col0 + lane] =
                    *reinterpret_cast<const uint16_t*>(buf + staged(r, lane >> 3) + (lane & 7) * 2);
    }
}

// Walks the tiles in bands of `band` row tiles, down the band first: the tiles in flight then share few rows of x
// and few of w, and a band's rows of x stay in L2 while all of w passes by.
__device__ __forceinline__ void tile_at(const LinearParams& p, int t, int& tm, int& tn) {
    const int per_band = p.band * p.tiles_n;
    const int b = t / per_band, in = t - b * per_band;
    const int rows = min(p.band, p.tiles_m - b * p.band);
    tn = in / rows;
    tm = b * p.band + in - tn * rows;
}

template <bool kFp8>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPairThreads, 1)
    linear_pair_kernel(const __grid_constant__ LinearParams p) {
    extern __shared__ char smem_raw[];
    char* smem = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    char* staging = smem + kPairStages * kPairStageBytes;
    char* ctl = staging + 8 * kStagingBytes;
    const uint32_t bars = smem_u32(ctl);
    const uint32_t full = bars, empty = bars + 8 * kPairStages, acc_full = bars + 16 * kPairStages, acc_empty = acc_full + 16;
    const uint32_t drain = acc_empty + 16;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(ctl + 16 * kPairStages + 40);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);  // [0] raised, [1] site
    int* dead = const_cast<int*>(abort_flag) + 2;                               // this block's view of the status word
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank();
    const uint32_t limit = p.wait_limit_us;

    if (threadIdx.x == 0) {
        for (int i = 0; i < kPairStages; ++i) {
            mbar_init(full + 8 * i, 1);
            mbar_init(empty + 8 * i, 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(acc_full + 8 * i, 1);
            mbar_init(acc_empty + 8 * i, 16);
        }
        mbar_init(drain, 1);
        fence_mbar_init();
        abort_flag[0] = abort_flag[1] = 0;
        tma_prefetch_desc(&p.tm_x);
        tma_prefetch_desc(&p.tm_w);
        *dead = p.status && *reinterpret_cast<volatile int*>(p.status) != 0;
    }
    if (warp == 2) {
        tmem_alloc_pair(smem_u32(tmem_slot), 512);
        tmem_relinquish_pair();
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    // Both blocks take the same decision, from what both of them saw.
    const bool gave_up_before = (*dead | cluster_load_i32(cluster_map(smem_u32(dead), rank ^ 1))) != 0;
    const int tiles = p.tiles_m * p.tiles_n;
    const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;

    if (warp == 0) {
        if (lane == 0 && !gave_up_before && !p.test_withhold) {
            const uint32_t ring = smem_u32(smem);
            const uint32_t w_bytes = static_cast<uint32_t>(p.tile_n / 2) * kStepBytes;
            const uint32_t full0 = cluster_map(full, 0);  // the pair's barriers are those of its first block
            int stage = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int t = pair; t < tiles && ok; t += pairs) {
                int tm, tn;
                tile_at(p, t, tm, tn);
                const int row_x = tm * 256 + static_cast<int>(rank) * 128;
                const int row_w = tn * p.tile_n + static_cast<int>(rank) * (p.tile_n / 2);
                for (int ks = 0; ks < p.k_steps; ++ks) {
                    if (!mbar_wait(empty + 8 * stage, phase ^ 1, abort_flag, 1, limit)) {
                        ok = false;
                        break;
                    }
                    if (rank == 0) mbar_arrive_expect_tx(full + 8 * stage, 2 * (kRowTile + w_bytes));
                    const uint32_t dst = ring + stage * kPairStageBytes;
                    tma_load_4d_pair(dst, &p.tm_x, full0 + 8 * stage, ks * p.k_step_elems, row_x, 0, 0);
                    tma_load_4d_pair(dst + kRowTile, &p.tm_w, full0 + 8 * stage, ks * p.k_step_elems, row_w, 0, 0);
                    if (++stage == kPairStages) {
                        stage = 0;
                        phase ^= 1;
                    }
                }
            }
            // Nothing of this block's may be in flight when it exits: every stage that was filled has been
            // consumed (the release also tells that the loads landed), or, after a wait gave up, has landed.
            // (The barriers of a stage that was never filled let both waits pass.)
            for (int i = 0; i < kPairStages; ++i) {
                if (ok) {
                    ok = mbar_wait(empty + 8 * stage, phase ^ 1, abort_flag, 2, limit);
                } else if (rank == 0) {
                    mbar_wait_drain(full + 8 * stage, phase ^ 1);
                }
                if (++stage == kPairStages) {
                    stage = 0;
                    phase ^= 1;
                }
            }
        }
    } else if (warp == 1) {
        if (lane == 0 && rank == 0 && !gave_up_before) {
            const uint32_t ring = smem_u32(smem);
            int stage = 0, acc = 0;
            uint32_t phase = 0, acc_phase = 0;
            bool ok = true;
            for (int t = pair; t < tiles && ok; t += pairs) {
                if (!mbar_wait(acc_empty + 8 * acc, acc_phase ^ 1, abort_flag, 3, limit)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const uint32_t d = tmem + acc * 256;
                for (int ks = 0; ks < p.k_steps; ++ks) {
                    if (!mbar_wait(full + 8 * stage, phase, abort_flag, 4, limit)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t a = desc_lo(ring + stage * kPairStageBytes, 16);
                    const uint32_t b = desc_lo(ring + stage * kPairStageBytes + kRowTile, 16);
#pragma unroll
                    for (int i = 0; i < 4; ++i)  // 32 bytes of k per MMA
                        umma_ss_pair<kFp8>(d, a + 2 * i, b + 2 * i, kDescHiSbo1024, p.idesc, (ks | i) != 0);
                    umma_commit_pair(empty + 8 * stage);
                    if (++stage == kPairStages) {
                        stage = 0;
                        phase ^= 1;
                    }
                }
                if (ok) umma_commit_pair(acc_full + 8 * acc);
                if ((acc ^= 1) == 0) acc_phase ^= 1;
            }
            if (!ok) {  // tensor memory and the operands stay until the MMAs that were issued are over
                umma_commit_pair(drain);
                mbar_wait_drain(drain, 0);
            }
        }
    } else if (warp >= 4) {
        const Epilogue& e = p.e;
        const int quarter = warp & 3, half = (warp - 4) >> 2;
        char* buf = staging + (warp - 4) * kStagingBytes;
        const uint32_t acc_empty0 = cluster_map(acc_empty, 0);
        int acc = 0;
        uint32_t acc_phase = 0;
        bool ok = !gave_up_before;
        const int chunks = p.tile_n / 32;
        for (int t = pair; t < tiles; t += pairs) {
            int tm, tn;
            tile_at(p, t, tm, tn);
            const int row0 = tm * 256 + static_cast<int>(rank) * 128 + quarter * 32;
            const int row = row0 + lane;
            const bool live = row < e.m;
            float xs = 1.0f;
            if (kFp8 && live) xs = __ldg(e.x_scale + static_cast<int64_t>(row) * e.x_scale_step);
            const int64_t gate_at = e.gate && live ? static_cast<int64_t>(static_cast<uint32_t>(row) / e.rows_per_gate) * e.gate_stride : 0;
            if (ok) ok = mbar_wait(acc_full + 8 * acc, acc_phase, abort_flag, 5, limit);
            ok = __all_sync(0xffffffffu, ok);
            tc_fence_after();
            for (int c = half; c < chunks; c += 2) {
                const int col0 = tn * p.tile_n + c * 32;
                uint32_t acc_bits[32];
                if (ok) {
                    tmem_ld32(tmem + (static_cast<uint32_t>(quarter * 32) << 16) + acc * 256 + c * 32, acc_bits);
                    if (e.residual && col0 < e.n)
                        stage_in(buf, static_cast<const uint16_t*>(e.residual), e.residual_stride, row0, col0, e.m, e.n,
                                 e.wide_residual, lane);
                    tmem_wait_ld();
                } else {
#pragma unroll
                    for (int i = 0; i < 32; ++i) acc_bits[i] = 0x7fc00000u;  // NaN: never plausible numbers
                }
                if (col0 >= e.n) continue;
                __syncwarp();
                uint4 old[4];
                if (e.residual) {
#pragma unroll
                    for (int q = 0; q < 4; ++q) old[q] = *reinterpret_cast<const uint4*>(buf + staged(lane, q));
                    __syncwarp();
                }
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int col = col0 + q * 8;
                    float v[8], f[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(acc_bits[q * 8 + i]);
                    if constexpr (kFp8) {
                        if (e.w_scale_step) {
                            load_cols8(e.w_scale, MINDIESD_FP32, 0, col, e.n, e.wide_cols, f);
#pragma unroll
                            for (int i = 0; i < 8; ++i) v[i] *= xs * f[i];
                        } else {
                            const float s = xs * __ldg(e.w_scale);
#pragma unroll
                            for (int i = 0; i < 8; ++i) v[i] *= s;
                        }
                    }
                    if (e.bias) {
                        load_cols8(e.bias, e.bias_type, 0, col, e.n, e.wide_cols, f);
#pragma unroll
                        for (int i = 0; i < 8; ++i) v[i] += f[i];
                    }
                    activate(v, e.act);
                    if (e.gate) {
                        load_cols8(e.gate, e.gate_type, gate_at, col, e.n, e.wide_cols, f);
#pragma unroll
                        for (int i = 0; i < 8; ++i) v[i] *= f[i];
                    }
                    if (e.residual) {
                        const uint32_t w[4] = {old[q].x, old[q].y, old[q].z, old[q].w};
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            float lo, hi;
                            unpack_pair(w[i], e.out_fp16, lo, hi);
                            v[2 * i] += lo;
                            v[2 * i + 1] += hi;
                        }
                    }
                    *reinterpret_cast<uint4*>(buf + staged(lane, q)) =
                        make_uint4(pack_pair(v[0], v[1], e.out_fp16), pack_pair(v[2], v[3], e.out_fp16),
                                   pack_pair(v[4], v[5], e.out_fp16), pack_pair(v[6], v[7], e.out_fp16));
                }
                __syncwarp();
                stage_out(buf, static_cast<uint16_t*>(e.out), e.out_stride, row0, col0, e.m, e.n, e.wide_out, lane);
                __syncwarp();
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0 && ok) mbar_arrive_cluster(acc_empty0 + 8 * acc);
            if ((acc ^= 1) == 0) acc_phase ^= 1;
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();  // neither block's memory goes while the other may still use it
    tc_fence_after();
    if (warp == 2) tmem_dealloc_pair(tmem, 512);
    if (threadIdx.x == 0) report(p, abort_flag);
}

// ---- few rows ----------------------------------------------------------------------------------------------

constexpr int kSwapThreads = 192;  // warps: 0 loader, 1 tensor memory + MMA, 2..5 epilogue
constexpr int kSwapMaxStages = 16;
constexpr int kSwapCtlBytes = 16 * kSwapMaxStages + 64;

template <bool kFp8>
__global__ void __launch_bounds__(kSwapThreads) linear_swap_kernel(const __grid_constant__ LinearParams p) {
    extern __shared__ char smem_raw[];
    char* smem = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    const uint32_t stage_bytes = kRowTile + static_cast<uint32_t>(p.tile_n) * kStepBytes;
    char* ctl = smem + p.stages * stage_bytes;
    const uint32_t full = smem_u32(ctl), empty = full + 8 * kSwapMaxStages, done = empty + 8 * kSwapMaxStages;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(ctl + 16 * kSwapMaxStages + 8);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = blockIdx.x;  // the cluster spans the x dimension of the grid
    const uint32_t limit = p.wait_limit_us;
    const int row_w = blockIdx.y * 128, row_x = blockIdx.z * p.tile_n;
    const int ks0 = static_cast<int>(static_cast<int64_t>(p.k_steps) * rank / p.split);
    const int ks1 = static_cast<int>(static_cast<int64_t>(p.k_steps) * (rank + 1) / p.split);

    if (threadIdx.x == 0) {
        for (int i = 0; i < p.stages; ++i) {
            mbar_init(full + 8 * i, 1);
            mbar_init(empty + 8 * i, 1);
        }
        mbar_init(done, 1);
        fence_mbar_init();
        abort_flag[0] = abort_flag[1] = 0;
        tma_prefetch_desc(&p.tm_x);
        tma_prefetch_desc(&p.tm_w);
    }
    if (warp == 1) {
        tmem_alloc(smem_u32(tmem_slot), p.tmem_cols);
        tmem_relinquish();
    }
    tc_fence_before();
    const bool dead = __syncthreads_or(threadIdx.x == 0 && p.status && *reinterpret_cast<volatile int*>(p.status) != 0);
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    bool ok = !dead;

    if (warp == 0) {
        if (lane == 0 && ok && !p.test_withhold) {
            const uint32_t ring = smem_u32(smem);
            int stage = 0;
            uint32_t phase = 0;
            for (int ks = ks0; ks < ks1; ++ks) {
                if (!mbar_wait(empty + 8 * stage, phase ^ 1, abort_flag, 6, limit)) {
                    ok = false;
                    break;
                }
                mbar_arrive_expect_tx(full + 8 * stage, stage_bytes);
                const uint32_t dst = ring + stage * stage_bytes;
                tma_load_4d(dst, &p.tm_w, full + 8 * stage, ks * p.k_step_elems, row_w, 0, 0);
                tma_load_4d(dst + kRowTile, &p.tm_x, full + 8 * stage, ks * p.k_step_elems, row_x, 0, 0);
                if (++stage == p.stages) {
                    stage = 0;
                    phase ^= 1;
                }
            }
            if (!ok)  // a wait gave up: the block may not go on to reuse the ring before its copies have landed
                for (int i = 0; i < p.stages; ++i) {
                    mbar_wait_drain(full + 8 * stage, phase ^ 1);
                    if (++stage == p.stages) {
                        stage = 0;
                        phase ^= 1;
                    }
                }
        }
    } else if (warp == 1) {
        if (lane == 0 && ok) {
            const uint32_t ring = smem_u32(smem);
            int stage = 0;
            uint32_t phase = 0;
            for (int ks = ks0; ks < ks1; ++ks) {
                if (!mbar_wait(full + 8 * stage, phase, abort_flag, 7, limit)) break;
                tc_fence_after();
                const uint32_t a = desc_lo(ring + stage * stage_bytes, 16);
                const uint32_t b = desc_lo(ring + stage * stage_bytes + kRowTile, 16);
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    umma_ss_lohi<kFp8>(tmem, a + 2 * i, b + 2 * i, kDescHiSbo1024, p.idesc, (ks > ks0 || i) ? 1u : 0u);
                umma_commit(empty + 8 * stage);
                if (++stage == p.stages) {
                    stage = 0;
                    phase ^= 1;
                }
            }
            umma_commit(done);  // also after a wait that gave up: the MMAs that were issued must be over
            mbar_wait_drain(done, 0);
        }
    } else if (ok) {
        ok = mbar_wait(done, 0, abort_flag, 8, limit);
    }
    __syncwarp();
    // The loader's drain, the MMA thread's wait and the epilogue's wait are all over: the ring is free.
    ok = __syncthreads_and(ok && abort_flag[0] == 0);
    tc_fence_after();

    const Epilogue& e = p.e;
    const int quarter = warp & 3;
    const int channel = row_w + quarter * 32 + lane;  // warps 2..5 cover the four quarters of the 128 lanes
    const bool live = channel < e.n;
    const bool worker = warp >= 2;
    float bias = 0.0f, ws = 1.0f;
    if (worker && live) {
        if (e.bias) bias = load_any(e.bias, e.bias_type, channel);
        if (kFp8) ws = __ldg(e.w_scale + static_cast<int64_t>(channel) * e.w_scale_step);
    }
    auto finish = [&](float acc, int token) {
        const int64_t row = row_x + token;
        float v[1] = {acc};
        if (kFp8) v[0] *= __ldg(e.x_scale + row * e.x_scale_step) * ws;
        if (e.bias) v[0] += bias;
        activate(v, e.act);
        if (e.gate)
            v[0] *= load_any(e.gate, e.gate_type, static_cast<int64_t>(static_cast<uint32_t>(row) / e.rows_per_gate) * e.gate_stride + channel);
        if (e.residual) v[0] += load_any(e.residual, e.out_fp16 ? MINDIESD_FP16 : MINDIESD_BF16, row * e.residual_stride + channel);
        if (e.out_fp16) static_cast<__half*>(e.out)[row * e.out_stride + channel] = __float2half_rn(v[0]);
        else static_cast<__nv_bfloat16*>(e.out)[row * e.out_stride + channel] = __float2bfloat16_rn(v[0]);
    };
    const int tokens = min(p.tile_n, e.m - row_x);
    const float bad = __uint_as_float(0x7fc00000u);
    float* partial = reinterpret_cast<float*>(smem);  // [token][128]
    if (worker) {
        const int lane_at = quarter * 32 + lane;
        for (int c = 0; c < tokens; c += 8) {
            uint32_t r[8];
            if (ok) {
                tmem_ld8(tmem + (static_cast<uint32_t>(quarter * 32) << 16) + c, r);
                tmem_wait_ld();
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float v = ok ? __uint_as_float(r[i]) : bad;
                if (p.split > 1) partial[(c + i) * 128 + lane_at] = v;
                else if (live && c + i < tokens) finish(v, c + i);
            }
        }
        tc_fence_before();
    }
    __syncwarp();
    if (p.split > 1) {
        cluster_sync_all();
        if (worker) {
            const uint32_t mine = smem_u32(partial) + (quarter * 32 + lane) * 4;
            for (int t = rank; t < tokens; t += p.split) {
                float sum = 0.0f;
                for (int r = 0; r < p.split; ++r) sum += cluster_load_f32(cluster_map(mine + t * 512, r));
                if (live) finish(sum, t);
            }
        }
        __syncwarp();
        cluster_sync_all();  // the partials are read by the other blocks until here
    }
    __syncthreads();
    if (warp == 1) tmem_dealloc(tmem, p.tmem_cols);
    if (threadIdx.x == 0) report(p, abort_flag);
}

// ---- host --------------------------------------------------------------------------------------------------

constexpr int kSms = 148;
constexpr int kMaxSmem = 227 * 1024;

template <bool kFp8>
cudaError_t launch_pair(LinearParams& p, cudaStream_t stream) {
    cudaError_t err = cudaFuncSetAttribute(linear_pair_kernel<kFp8>, cudaFuncAttributeMaxDynamicSharedMemorySize, kPairSmem);
    if (err != cudaSuccess) return err;
    const int64_t tiles = static_cast<int64_t>(p.tiles_m) * p.tiles_n;
    const int pairs = static_cast<int>(tiles < kSms / 2 ? tiles : kSms / 2);
    linear_pair_kernel<kFp8><<<2 * pairs, kPairThreads, kPairSmem, stream>>>(p);
    return cudaGetLastError();
}

template <bool kFp8>
cudaError_t launch_swap(LinearParams& p, int smem, cudaStream_t stream) {
    cudaError_t err = cudaFuncSetAttribute(linear_swap_kernel<kFp8>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (err != cudaSuccess) return err;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(p.split, (p.e.n + 127) / 128, (p.e.m + p.tile_n - 1) / p.tile_n);
    cfg.blockDim = dim3(kSwapThreads, 1, 1);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = p.split;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, linear_swap_kernel<kFp8>, p);
}

}  // namespace
}  // namespace sdb

using namespace sdb;

extern "C" int mindiesd_linear_fwd(const mindiesd_linear_args* a, void* stream_) {
    if (!a || !a->x || !a->weight || !a->out) return MINDIESD_E_NULL;
    if (a->m <= 0 || a->n <= 0 || a->k <= 0) return MINDIESD_E_SHAPE;
    if (a->m > 0x7fff0000 || a->n > 0x7fff0000 || a->k > 0x7fff0000) return MINDIESD_E_CAPACITY;  // tile coordinates are 32-bit
    const bool fp8 = a->in_dtype == MINDIESD_E4M3;
    if (!fp8 && a->in_dtype != MINDIESD_BF16 && a->in_dtype != MINDIESD_FP16) return MINDIESD_E_DTYPE;
    if (a->out_dtype != MINDIESD_BF16 && a->out_dtype != MINDIESD_FP16) return MINDIESD_E_DTYPE;
    auto float_type = [](int t) { return t == MINDIESD_BF16 || t == MINDIESD_FP16 || t == MINDIESD_FP32; };
    if (a->bias && !float_type(a->bias_dtype)) return MINDIESD_E_DTYPE;
    if (a->gate && !float_type(a->gate_dtype)) return MINDIESD_E_DTYPE;
    if (fp8 && (!a->x_scale || !a->weight_scale)) return MINDIESD_E_NULL;
    if (!fp8 && (a->x_scale || a->weight_scale)) return MINDIESD_E_VALUE;
    if (a->activation < MINDIESD_ACT_NONE || a->activation > MINDIESD_ACT_GELU_TANH) return MINDIESD_E_VALUE;
    if (a->gate && a->rows_per_gate <= 0) return MINDIESD_E_VALUE;
    // Rows must not overlap (a stride of 0 would be one row seen many times: the tensor map cannot say that).
    auto rows_apart = [](int64_t stride, int64_t len, int64_t rows) { return rows <= 1 || stride >= len; };
    if (!rows_apart(a->x_stride, a->k, a->m) || !rows_apart(a->weight_stride, a->k, a->n) || !rows_apart(a->out_stride, a->n, a->m))
        return MINDIESD_E_STRIDE;
    if ((a->residual && a->residual_stride < 0) || (a->gate && a->gate_stride < 0)) return MINDIESD_E_STRIDE;
    auto aligned = [](const void* ptr, int bytes) { return reinterpret_cast<uintptr_t>(ptr) % bytes == 0; };
    if (!aligned(a->out, 2) || !aligned(a->residual, 2) || !aligned(a->x_scale, 4) || !aligned(a->weight_scale, 4)) return MINDIESD_E_STRIDE;
    if (a->bias && !aligned(a->bias, dtype_bytes(a->bias_dtype))) return MINDIESD_E_STRIDE;
    if (a->gate && !aligned(a->gate, dtype_bytes(a->gate_dtype))) return MINDIESD_E_STRIDE;

    const int eb = fp8 ? 1 : 2;
    LinearParams p = {};
    p.k_step_elems = kStepBytes / eb;
    p.k_steps = (a->k + p.k_step_elems - 1) / p.k_step_elems;
    Epilogue& e = p.e;
    e.bias = a->bias;
    e.residual = a->residual;
    e.gate = a->gate;
    e.x_scale = a->x_scale;
    e.w_scale = a->weight_scale;
    e.out = a->out;
    e.residual_stride = a->residual_stride;
    e.out_stride = a->m > 1 ? a->out_stride : a->n;
    e.gate_stride = a->gate_stride;
    e.rows_per_gate = a->gate ? static_cast<uint32_t>(a->rows_per_gate) : 1u;
    e.x_scale_step = a->x_scale_single ? 0 : 1;
    e.w_scale_step = a->weight_scale_single ? 0 : 1;
    e.bias_type = a->bias_dtype;
    e.gate_type = a->gate_dtype;
    e.out_fp16 = a->out_dtype == MINDIESD_FP16;
    e.act = a->activation;
    e.m = a->m;
    e.n = a->n;
    // 16-byte access: rows start on a 16-byte boundary and hold whole vectors.
    e.wide_out = aligned(a->out, 16) && e.out_stride % 8 == 0 && a->n % 8 == 0;
    e.wide_residual = a->residual && aligned(a->residual, 16) && a->residual_stride % 8 == 0 && a->n % 8 == 0;
    e.wide_cols = aligned(a->bias, 16) && aligned(a->gate, 16) && aligned(a->weight_scale, 16) &&
                  (!a->gate || (a->gate_stride * dtype_bytes(a->gate_dtype)) % 16 == 0);
    p.wait_limit_us = a->wait_limit_us ? a->wait_limit_us : kWaitLimitUs;
    p.test_withhold = a->test_withhold;
    p.status = device_status_word();
    const uint32_t fmt = a->in_dtype == MINDIESD_BF16 ? 1u : 0u;
    const int64_t xs[3] = {a->m > 1 ? a->x_stride : 16 * ((a->k + 15) / 16), 0, 0};
    const int64_t ws[3] = {a->n > 1 ? a->weight_stride : 16 * ((a->k + 15) / 16), 0, 0};
    const int64_t x_strides[3] = {xs[0], xs[0], xs[0]}, w_strides[3] = {ws[0], ws[0], ws[0]};
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    int rc;
    cudaError_t err;
    if (a->m <= 128) {
        p.tile_n = (a->m + 15) / 16 * 16;
        p.tmem_cols = p.tile_n <= 32 ? 32 : p.tile_n <= 64 ? 64 : 128;
        p.idesc = umma_idesc(fmt, 128, p.tile_n, false, false);
        const int stage_bytes = kRowTile + p.tile_n * kStepBytes;
        const int budget = 74 * 1024 - 1024 - kSwapCtlBytes;
        p.stages = budget / stage_bytes;
        if (p.stages > kSwapMaxStages) p.stages = kSwapMaxStages;
        if (p.stages < 4) p.stages = 4;
        const int smem = p.stages * stage_bytes + kSwapCtlBytes + 1024;
        const int blocks = (a->n + 127) / 128;
        const int slots = kSms * (kMaxSmem / (smem + 1024));
        p.split = 1;
        while (p.split < 8 && (p.split + 1) * blocks <= slots && p.k_steps >= 2 * (p.split + 1)) ++p.split;
        if ((rc = encode_tile_map(&p.tm_w, a->weight, a->in_dtype, a->k, a->n, 1, 1, w_strides, 128))) return rc;
        if ((rc = encode_tile_map(&p.tm_x, a->x, a->in_dtype, a->k, a->m, 1, 1, x_strides, p.tile_n))) return rc;
        if (blocks > 65535) return MINDIESD_E_CAPACITY;
        err = fp8 ? launch_swap<true>(p, smem, stream) : launch_swap<false>(p, smem, stream);
    } else {
        p.tile_n = 256;
        p.tiles_m = (a->m + 255) / 256;
        p.tiles_n = (a->n + p.tile_n - 1) / p.tile_n;
        if (static_cast<int64_t>(p.tiles_m) * p.tiles_n > 0x3fffffff) return MINDIESD_E_CAPACITY;
        p.band = 8;
        p.idesc = umma_idesc(fmt, 256, p.tile_n, false, false);
        if ((rc = encode_tile_map(&p.tm_x, a->x, a->in_dtype, a->k, a->m, 1, 1, x_strides, 128))) return rc;
        if ((rc = encode_tile_map(&p.tm_w, a->weight, a->in_dtype, a->k, a->n, 1, 1, w_strides, p.tile_n / 2))) return rc;
        err = fp8 ? launch_pair<true>(p, stream) : launch_pair<false>(p, stream);
    }
    return err == cudaSuccess ? MINDIESD_OK : static_cast<int>(err);
}
