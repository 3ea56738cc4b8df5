// Matrix product with its epilogue:  out = residual + gate * act(x w^T * scales + bias).
//   x [m, k], w [n, k] (both k-contiguous), bf16 / fp16 / e4m3 operands, fp32 accumulation, one rounding of the result.
//
// Two kernels.  Both stream 128-byte wide tiles of x and w through a ring of shared-memory stages filled by a TMA
// warp, and one warp issues tcgen05 MMAs into tensor memory.
//
// `linear_pair_kernel` (many rows): persistent, two thread blocks (a cluster on neighbouring SMs) work on one
// 256 x tile_n tile with two-SM MMAs, so each SM fetches 128 rows of x and only HALF of the tile's rows of w: 32 KB
// per 128 x 256 x 128-byte step.  Two accumulators of up to 256 columns: the epilogue of a tile (16 warps per block)
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

#include <algorithm>
#include <atomic>
#include <mutex>

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
    int out_piece, residual_piece;   // bytes of a row that can be moved at a time (piece_of)
    int wide_gate;                   // 16 of them
    int m, n;
};

struct LinearParams {
    alignas(64) CUtensorMap tm_x;
    alignas(64) CUtensorMap tm_w;
    Epilogue e;
    int k_steps, k_step_elems;
    int tile_n;                    // pair kernel: columns of a tile; swap kernel: tokens of a tile
    int tiles_m, tiles_n, band;    // pair kernel: tiles are walked in bands of `band` row tiles
    int stages;
    int tmem_cols, split;  // swap kernel
    uint32_t idesc;
    uint32_t wait_limit_us;
    int test_withhold;
    int* status;
};

__device__ __forceinline__ void prefetch_l2(const void* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }

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

template <bool kFp16, int kPairs>
__device__ __forceinline__ void pack_values(const uint64_t (&v)[kPairs], uint32_t (&w)[kPairs]) {
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
        float lo, hi;
        unpack2(v[i], lo, hi);
        w[i] = pack_pair(lo, hi, kFp16);
    }
}

// Eight consecutive column values of the gate row that starts at row_at.
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

__device__ __forceinline__ float rcp_approx(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint64_t both(float v) { return pack2(v, v); }

// v / (1 + 2^x) for a pair; the quotient is 0 where 2^x is above 2^126 (the reciprocal flushes there) or infinite.
__device__ __forceinline__ uint64_t over_one_plus_ex2(uint64_t v, uint64_t x) {
    float lo, hi;
    unpack2(x, lo, hi);
    const uint64_t d = add2(pack2(ex2_approx(lo), ex2_approx(hi)), both(1.0f));
    unpack2(d, lo, hi);
    return mul2(v, pack2(rcp_approx(lo), rcp_approx(hi)));
}

// gelu(v) = max(v, 0) - |v|/2 erfc(|v| / sqrt 2), which loses nothing for large negative v, for a pair of values.  With
// z = |v| / sqrt 2 and t = 1 / (1 + 0.45 z), erfc(z) = e^(-z^2) t P(t); P is the polynomial of degree 7 with the smallest
// largest relative error (3.5e-7) for z up to 14.2, found by linear programming.  Beyond, the product is 0.
// (CUDA's erfc, out of line: 9000 x 1024 x 5120 bf16 150 us, this 85, gelu_tanh 79; 9000 x 5120 x 5120 321 and 307.)
__device__ __forceinline__ uint64_t gelu_pair(uint64_t v) {
    constexpr float kP[8] = {0.253884882f, 0.254008859f, 0.225756422f, 0.196237445f, 0.0261506569f, 0.223944306f, -0.248876333f, 0.0688941106f};
    float lo, hi, x, y;
    unpack2(v, lo, hi);
    const uint64_t a = pack2(fminf(fabsf(lo), 20.0f), fminf(fabsf(hi), 20.0f));  // an infinity would give 0 * infinity
    unpack2(fma2(a, both(0.45f * 0.70710678f), both(1.0f)), x, y);
    const uint64_t t = pack2(rcp_approx(x), rcp_approx(y));
    uint64_t q = both(kP[7]);
#pragma unroll
    for (int i = 6; i >= 0; --i) q = fma2(q, t, both(kP[i]));
    unpack2(mul2(mul2(a, a), both(-0.5f * 1.4426950408889634f)), x, y);
    q = mul2(mul2(q, t), pack2(ex2_approx(x), ex2_approx(y)));
    return fma2(mul2(a, both(-0.5f)), q, pack2(lo < 0.0f ? 0.0f : lo, hi < 0.0f ? 0.0f : hi));  // a NaN stays
}

// The activations, on pairs of values, in the forms that keep their relative accuracy for large negative arguments, down to
// values of |v| 2^-126, which become 0 (silu below -87.3, gelu below -13.2, gelu_tanh below -10.0):
//   gelu(v) = v/2 erfc(-v / sqrt 2) (gelu_pair),  silu(v) = v / (1 + e^-v),
//   gelu_tanh(v) = v/2 (1 + tanh u) = v / (1 + e^-2u),  u = sqrt(2/pi) (v + 0.044715 v^3).
template <int kPairs>
__device__ __forceinline__ void activate(uint64_t (&v)[kPairs], int act) {
    constexpr float kLog2e = 1.4426950408889634f;
    constexpr float kU1 = -2.0f * 0.7978845608028654f * kLog2e, kU3 = kU1 * 0.044715f;
    switch (act) {
        case kRelu:
#pragma unroll
            for (int i = 0; i < kPairs; ++i) {
                float lo, hi;
                unpack2(v[i], lo, hi);
                v[i] = pack2(lo < 0.0f ? 0.0f : lo, hi < 0.0f ? 0.0f : hi);  // a NaN stays
            }
            break;
        case kSilu:
#pragma unroll
            for (int i = 0; i < kPairs; ++i) v[i] = over_one_plus_ex2(v[i], mul2(v[i], both(-kLog2e)));
            break;
        case kGelu:
#pragma unroll
            for (int i = 0; i < kPairs; ++i) v[i] = gelu_pair(v[i]);
            break;
        case kGeluTanh:
#pragma unroll
            for (int i = 0; i < kPairs; ++i)
                v[i] = over_one_plus_ex2(v[i], mul2(v[i], fma2(mul2(v[i], v[i]), both(kU3), both(kU1))));
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

constexpr int kEpilogueWarps = 16;
constexpr int kPairThreads = 128 + 32 * kEpilogueWarps;  // warps: 0 loader, 1 MMA, 2 tensor memory, 3 idle, 4.. epilogue
constexpr int kSub = 2;  // swap kernel: k steps per ring stage, one barrier round trip and one commit for eight MMAs
constexpr int kRingBytes = 6 * 2 * kRowTile;  // pair kernel: three stages of 256-column tiles, more of narrower ones
constexpr int kPairMaxStages = 8;
// The epilogue works in units of 32 rows x 16 columns.  Four warps share a quarter of the tile's rows and take its
// units in turn: with two warps of 32-column units a 256-column tile left 4 us of epilogue after its last MMA, and
// the latency of one warp's instructions, not their number, was what it waited for.
constexpr int kUnit = 16;
constexpr int kUnitWarps = kEpilogueWarps / 4;
constexpr int kMaxUnits = 256 / kUnit / kUnitWarps;  // of one warp in one tile
constexpr int kStagingBytes = 32 * kUnit * 2;        // per warp: one unit of two-byte values
constexpr int kColsBytes = 3 * kMaxUnits * kUnit * 4;  // per warp: bias, weight scale and gate of its columns as fp32
constexpr int kPairSmem = kRingBytes + kEpilogueWarps * (kStagingBytes + kColsBytes) + 256 + 1024;
static_assert(kPairSmem <= 227 * 1024, "shared memory of the pair kernel");

// Offset of 16-byte piece c of row r in a warp's staging buffer; the exclusive or keeps both the row-wise writes and
// the piece-wise reads free of bank conflicts.
__device__ __forceinline__ uint32_t staged(int r, int c) { return r * 32 + ((c ^ ((r >> 2) & 1)) << 4); }

// A lane's share of a unit on its way through the staging buffer: 8 columns of rows lane/2 and lane/2 + 16 of the warp's 32.
struct UnitAt {
    const uint16_t* p[2];
    bool live[2];  // the rows exist
    __device__ __forceinline__ UnitAt(const void* base, int64_t stride, int row0, int m, int lane) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int r = row0 + i * 16 + (lane >> 1);
            live[i] = r < m;
            p[i] = static_cast<const uint16_t*>(base) + static_cast<int64_t>(r) * stride + (lane & 1) * 8;
        }
    }
};

// 32 bytes of a row that starts on a multiple of 32.
__device__ __forceinline__ void load_row32(uint32_t (&w)[8], const uint16_t* p) {
    asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
                 : "l"(p)
                 : "memory");
}
__device__ __forceinline__ void store_row32(uint16_t* p, const uint32_t (&w)[8]) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]),
                 "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
}

// `piece`: 16 or 8 bytes where every row starts on a multiple of that and holds whole ones, else 2.  Rows of an odd
// width start on 4 bytes and between them in turn; the words of the latter are shifted by one element.
__device__ __forceinline__ void fetch_unit(uint32_t (&words)[8], const UnitAt& at, int col0, int n, int piece, int lane) {
    const int left = n - col0 - (lane & 1) * 8;  // columns of this lane that exist
    uint4 v[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        if (!at.live[i] || left <= 0) continue;
        const uint16_t* p = at.p[i] + col0;
        if (piece == 16) {
            v[i] = __ldg(reinterpret_cast<const uint4*>(p));
        } else if (piece == 8) {
            const uint2 lo = __ldg(reinterpret_cast<const uint2*>(p));
            const uint2 hi = left > 4 ? __ldg(reinterpret_cast<const uint2*>(p) + 1) : make_uint2(0, 0);
            v[i] = make_uint4(lo.x, lo.y, hi.x, hi.y);
        } else if (left >= 8) {
            const bool odd = reinterpret_cast<uintptr_t>(p) & 2;
            const uint32_t* q = reinterpret_cast<const uint32_t*>(p + odd);
            const uint32_t a = __ldg(q), b = __ldg(q + 1), c = __ldg(q + 2);
            if (odd) {
                const uint32_t first = __ldg(p), last = __ldg(p + 7);
                v[i] = make_uint4(first | (a << 16), (a >> 16) | (b << 16), (b >> 16) | (c << 16), (c >> 16) | (last << 16));
            } else {
                v[i] = make_uint4(a, b, c, __ldg(q + 3));
            }
        } else {
            uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (j < left) w[j >> 1] |= static_cast<uint32_t>(p[j]) << ((j & 1) * 16);
            v[i] = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        words[4 * i] = v[i].x;
        words[4 * i + 1] = v[i].y;
        words[4 * i + 2] = v[i].z;
        words[4 * i + 3] = v[i].w;
    }
}
// Turns what fetch_unit loaded into this lane's row of the unit, through the warp's staging buffer.
__device__ __forceinline__ void turn_unit(char* buf, uint32_t (&w)[8], int lane) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
        *reinterpret_cast<uint4*>(buf + staged(i * 16 + (lane >> 1), lane & 1)) = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
    __syncwarp();
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        const uint4 v = *reinterpret_cast<const uint4*>(buf + staged(lane, q));
        w[4 * q] = v.x;
        w[4 * q + 1] = v.y;
        w[4 * q + 2] = v.z;
        w[4 * q + 3] = v.w;
    }
    __syncwarp();
}

// Writes a warp's staging buffer to the output where the rows' pieces are smaller than 32 bytes: 16 rows of 32 bytes at a time,
// or fewer rows in smaller pieces (9000 x 256 x n bf16, single elements 94 us: n 5128 55 us, 5124 60 in pieces of 8 bytes,
// 5122 84 and 5121 92 in words; 5120, where a lane stores its own 32 bytes, 46, and 52 through this buffer).
__device__ __forceinline__ void stage_out(const char* buf, const UnitAt& at, const Epilogue& e, int row0, int col0, int lane) {
    if (e.out_piece == 16) {
        if (col0 + (lane & 1) * 8 < e.n) {
#pragma unroll
            for (int i = 0; i < 2; ++i)
                if (at.live[i])
                    *reinterpret_cast<uint4*>(const_cast<uint16_t*>(at.p[i]) + col0) =
                        *reinterpret_cast<const uint4*>(buf + staged(i * 16 + (lane >> 1), lane & 1));
        }
        return;
    }
    uint16_t* const g = static_cast<uint16_t*>(e.out) + static_cast<int64_t>(row0) * e.out_stride + col0;
    if (e.out_piece == 8) {
        const int c = (lane & 3) * 4;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = i * 8 + (lane >> 2);
            if (row0 + r < e.m && col0 + c < e.n)
                *reinterpret_cast<uint2*>(g + r * e.out_stride + c) = *reinterpret_cast<const uint2*>(buf + staged(r, c >> 3) + (c & 4) * 2);
        }
    } else if (col0 + kUnit <= e.n) {
        // Word c of every fourth row: whether its rows start between words does not change from one to the next.
        const int c = lane & 7, r0 = lane >> 3, c1 = (c + 1) & 7;
        uint16_t* p = g + r0 * e.out_stride + c * 2;
        const uint32_t odd = (reinterpret_cast<uintptr_t>(p) & 2) / 2;
        p += odd;
        const int live = c == 7 && odd ? 0 : e.m - row0 - r0;  // rows of this lane lie below it
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const char* row = buf + i * 128 + r0 * 32;
            const uint32_t lo = *reinterpret_cast<const uint32_t*>(row + ((((c >> 2) ^ i) & 1) << 4) + (c & 3) * 4);
            const uint32_t hi = *reinterpret_cast<const uint32_t*>(row + ((((c1 >> 2) ^ i) & 1) << 4) + (c1 & 3) * 4);
            if (i * 4 < live) *reinterpret_cast<uint32_t*>(p) = __funnelshift_r(lo, hi, odd * 16);
            p += 4 * e.out_stride;
        }
        uint16_t* ends = g + lane * e.out_stride;
        if (row0 + lane < e.m && (reinterpret_cast<uintptr_t>(ends) & 2)) {  // what the words leave of such a row
            ends[0] = *reinterpret_cast<const uint16_t*>(buf + staged(lane, 0));
            ends[15] = *reinterpret_cast<const uint16_t*>(buf + staged(lane, 1) + 14);
        }
    } else {
        const int c = lane & 15;
#pragma unroll 4
        for (int i = 0; i < 16; ++i) {
            const int r = i * 2 + (lane >> 4);
            if (row0 + r < e.m && col0 + c < e.n)
                g[r * e.out_stride + c] = *reinterpret_cast<const uint16_t*>(buf + staged(r, c >> 3) + (c & 7) * 2);
        }
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

// kSteps: k steps per ring stage (pair_sub).
template <bool kFp8, int kSteps>
__global__ void __launch_bounds__(kPairThreads, 1) linear_pair_kernel(const __grid_constant__ LinearParams p) {
    extern __shared__ char smem_raw[];
    char* smem = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    char* staging = smem + kRingBytes;
    char* columns = staging + kEpilogueWarps * kStagingBytes;
    char* ctl = columns + kEpilogueWarps * kColsBytes;
    const uint32_t bars = smem_u32(ctl);
    const uint32_t full = bars, empty = bars + 8 * kPairMaxStages, acc_full = bars + 16 * kPairMaxStages, acc_empty = acc_full + 16;
    const uint32_t drain = acc_empty + 16;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(ctl + 16 * kPairMaxStages + 40);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);  // [0] raised, [1] site
    int* dead = const_cast<int*>(abort_flag) + 2;                               // this block's view of the status word
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank();
    const uint32_t limit = p.wait_limit_us;

    if (threadIdx.x == 0) {
        for (int i = 0; i < p.stages; ++i) {
            mbar_init(full + 8 * i, 1);
            mbar_init(empty + 8 * i, 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(acc_full + 8 * i, 1);
            mbar_init(acc_empty + 8 * i, 2 * kEpilogueWarps);
        }
        mbar_init(drain, 1);
        fence_mbar_init();
        abort_flag[0] = abort_flag[1] = 0;
        tma_prefetch_desc(&p.tm_x);
        tma_prefetch_desc(&p.tm_w);
    }
    allow_next_kernel();
    if (warp == 2) {
        tmem_alloc_pair(smem_u32(tmem_slot), 512);
        tmem_relinquish_pair();
    }
    wait_for_kernels_before();
    if (threadIdx.x == 0) *dead = p.status && *reinterpret_cast<volatile int*>(p.status) != 0;
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    // Both blocks take the same decision, from what both of them saw.
    const bool gave_up_before = (*dead | cluster_load_i32(cluster_map(smem_u32(dead), rank ^ 1))) != 0;
    const int tiles = p.tiles_m * p.tiles_n;
    const uint32_t step_bytes = kRowTile + static_cast<uint32_t>(p.tile_n / 2) * kStepBytes;  // of one block
    const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;

    if (warp == 0) {
        if (!gave_up_before && !p.test_withhold) {
            const bool one = elect_one();
            const uint32_t ring = smem_u32(smem);
            const uint32_t full0 = cluster_map(full, 0);  // the pair's barriers are those of its first block
            int stage = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int t = pair; t < tiles && ok; t += pairs) {
                int tm, tn;
                tile_at(p, t, tm, tn);
                const int row_x = tm * 256 + static_cast<int>(rank) * 128;
                const int row_w = tn * p.tile_n + static_cast<int>(rank) * (p.tile_n / 2);
                for (int ks = 0; ks < p.k_steps; ks += kSteps) {
                    ok = mbar_wait_warp(empty + 8 * stage, phase ^ 1, abort_flag, 1, limit);
                    if (!ok) break;
                    const int subs = min(kSteps, p.k_steps - ks);
                    if (one) {
                        if (rank == 0) mbar_arrive_expect_tx(full + 8 * stage, subs * 2 * step_bytes);
                        uint32_t dst = ring + stage * kSteps * step_bytes;
                        for (int j = 0; j < subs; ++j, dst += step_bytes) {
                            tma_load_4d_pair(dst, &p.tm_x, full0 + 8 * stage, (ks + j) * p.k_step_elems, row_x, 0, 0);
                            tma_load_4d_pair(dst + kRowTile, &p.tm_w, full0 + 8 * stage, (ks + j) * p.k_step_elems, row_w, 0, 0);
                        }
                    }
                    if (++stage == p.stages) {
                        stage = 0;
                        phase ^= 1;
                    }
                }
            }
            // Nothing of this block's may be in flight when it exits: every stage that was filled has been
            // consumed (the release also tells that the loads landed), or, after a wait gave up, has landed.
            // (The barriers of a stage that was never filled let both waits pass.)
            for (int i = 0; i < p.stages; ++i) {
                if (ok) {
                    ok = mbar_wait_warp(empty + 8 * stage, phase ^ 1, abort_flag, 2, limit);
                } else if (rank == 0) {
                    mbar_wait_drain(full + 8 * stage, phase ^ 1);
                }
                if (++stage == p.stages) {
                    stage = 0;
                    phase ^= 1;
                }
            }
        }
    } else if (warp == 1) {
        if (rank == 0 && !gave_up_before) {
            const bool one = elect_one();
            const uint32_t ring = smem_u32(smem);
            int stage = 0, acc = 0;
            uint32_t phase = 0, acc_phase = 0;
            bool ok = true;
            for (int t = pair; t < tiles && ok; t += pairs) {
                ok = mbar_wait_warp(acc_empty + 8 * acc, acc_phase ^ 1, abort_flag, 3, limit);
                if (!ok) break;
                tc_fence_after();
                const uint32_t d = tmem + acc * 256;
                for (int ks = 0; ks < p.k_steps; ks += kSteps) {
                    ok = mbar_wait_warp(full + 8 * stage, phase, abort_flag, 4, limit);
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t a = desc_lo(ring + stage * kSteps * step_bytes, 16);
                    const uint32_t b = desc_lo(ring + stage * kSteps * step_bytes + kRowTile, 16);
                    if (one) {
#pragma unroll
                        for (int j = 0; j < kSteps; ++j) {
                            if (ks + j >= p.k_steps) break;
#pragma unroll
                            for (int i = 0; i < 4; ++i)  // 32 bytes of k per MMA
                                umma_ss_pair<kFp8>(d, a + j * (step_bytes >> 4) + 2 * i, b + j * (step_bytes >> 4) + 2 * i,
                                                   kDescHiSbo1024, p.idesc, (ks | j | i) != 0);
                        }
                        umma_commit_pair(empty + 8 * stage);
                        if (ks + kSteps >= p.k_steps) umma_commit_pair(acc_full + 8 * acc);
                    }
                    __syncwarp();
                    if (++stage == p.stages) {
                        stage = 0;
                        phase ^= 1;
                    }
                }
                if ((acc ^= 1) == 0) acc_phase ^= 1;
            }
            if (!ok) {  // tensor memory and the operands stay until the MMAs that were issued are over
                if (one) umma_commit_pair(drain);
                mbar_wait_drain(drain, 0);
            }
        }
    } else if (warp >= 4) {
        const Epilogue& e = p.e;
        const int quarter = warp & 3, turn = (warp - 4) >> 2;  // rows of the tile, first unit of this warp
        char* buf = staging + (warp - 4) * kStagingBytes;
        constexpr int kCols = kMaxUnits * kUnit;
        float* cols = reinterpret_cast<float*>(columns + (warp - 4) * kColsBytes);  // [bias | weight scale | gate][kCols]
        const uint32_t acc_empty0 = cluster_map(acc_empty, 0);
        const uint16_t* residual = static_cast<const uint16_t*>(e.residual);
        uint32_t ahead[kUnit / 2];  // the residual of the next unit: of this lane's row, or to be passed through shared memory
        int acc = 0;
        uint32_t acc_phase = 0;
        bool ok = !gave_up_before;
        const int units = p.tile_n / kUnit;
        for (int t = pair; t < tiles; t += pairs) {
            int tm, tn;
            tile_at(p, t, tm, tn);
            const int row0 = tm * 256 + static_cast<int>(rank) * 128 + quarter * 32;
            const int row = row0 + lane;
            const bool live = row < e.m;
            const UnitAt out_at(e.out, e.out_stride, row0, e.m, lane), residual_at(e.residual, e.residual_stride, row0, e.m, lane);
            float xs = 1.0f;
            if (kFp8 && live) xs = __ldg(e.x_scale + static_cast<int64_t>(row) * e.x_scale_step);
            // What the columns of this warp need is fetched while the MMAs of the tile still run.  The gate's row is
            // taken along where all rows of the warp share it (a sample's boundary can fall between them).
            const int64_t gate_at = e.gate && live ? static_cast<int64_t>(static_cast<uint32_t>(row) / e.rows_per_gate) * e.gate_stride : 0;
            const int64_t gate_first = __shfl_sync(0xffffffffu, gate_at, 0);
            const bool shared_gate = e.gate && __all_sync(0xffffffffu, !live || gate_at == gate_first);
            __syncwarp();
            float b2[kCols / 32] = {}, s2[kCols / 32] = {}, g2[kCols / 32] = {};  // all loads first: one trip to L2, not one for each
#pragma unroll
            for (int i = 0; i < kCols / 32; ++i) {
                const int u = turn + kUnitWarps * (2 * i + (lane >> 4)), col = tn * p.tile_n + u * kUnit + (lane & 15);
                if (u >= units || col >= e.n) continue;
                if (e.bias) b2[i] = load_any(e.bias, e.bias_type, col);
                if (kFp8) s2[i] = __ldg(e.w_scale + static_cast<int64_t>(col) * e.w_scale_step);
                if (shared_gate) g2[i] = load_any(e.gate, e.gate_type, gate_first + col);
            }
#pragma unroll
            for (int i = 0; i < kCols / 32; ++i) {
                cols[i * 32 + lane] = b2[i];
                if (kFp8) cols[kCols + i * 32 + lane] = s2[i];
                cols[2 * kCols + i * 32 + lane] = g2[i];
            }
            if (e.residual && live)  // its way from memory to L2 also runs under the MMAs
                for (int u = turn; u < units; u += kUnitWarps)
                    prefetch_l2(residual + static_cast<int64_t>(row) * e.residual_stride + min(tn * p.tile_n + u * kUnit, e.n - 1));
            __syncwarp();
            uint16_t* const out_row = static_cast<uint16_t*>(e.out) + static_cast<int64_t>(row) * e.out_stride;
            // Values of a unit's columns in this lane's row (the j-th unit of the warp), from accumulator to output.
            auto finish = [&](uint64_t (&v)[kUnit / 2], const uint32_t (&old)[kUnit / 2], int j, int col0) {
                const ulonglong2* at = reinterpret_cast<const ulonglong2*>(cols + j * kUnit);  // two pairs of columns per load
                if constexpr (kFp8) {  // one scale after the other: their product alone may be out of range
#pragma unroll
                    for (int i = 0; i < kUnit / 4; ++i) {
                        const ulonglong2 f = at[kCols / 4 + i];
                        v[2 * i] = mul2(mul2(v[2 * i], both(xs)), f.x);
                        v[2 * i + 1] = mul2(mul2(v[2 * i + 1], both(xs)), f.y);
                    }
                }
                if (e.bias) {
#pragma unroll
                    for (int i = 0; i < kUnit / 4; ++i) {
                        const ulonglong2 f = at[i];
                        v[2 * i] = add2(v[2 * i], f.x);
                        v[2 * i + 1] = add2(v[2 * i + 1], f.y);
                    }
                }
                activate(v, e.act);
                if (shared_gate) {
#pragma unroll
                    for (int i = 0; i < kUnit / 4; ++i) {
                        const ulonglong2 f = at[kCols / 2 + i];
                        v[2 * i] = mul2(v[2 * i], f.x);
                        v[2 * i + 1] = mul2(v[2 * i + 1], f.y);
                    }
                } else if (e.gate) {
#pragma unroll
                    for (int q = 0; q < kUnit / 8; ++q) {
                        float f[8];
                        load_cols8(e.gate, e.gate_type, gate_at, col0 + q * 8, e.n, e.wide_gate, f);
#pragma unroll
                        for (int i = 0; i < 4; ++i) v[q * 4 + i] = mul2(v[q * 4 + i], pack2(f[2 * i], f[2 * i + 1]));
                    }
                }
                if (e.residual) {
#pragma unroll
                    for (int i = 0; i < kUnit / 2; ++i) {
                        float lo, hi;
                        unpack_pair(old[i], e.out_fp16, lo, hi);
                        v[i] = add2(v[i], pack2(lo, hi));
                    }
                }
                uint32_t w[kUnit / 2];
                if (e.out_fp16) pack_values<true>(v, w);
                else pack_values<false>(v, w);
                if (e.out_piece == 32) {
                    if (live && col0 < e.n) store_row32(out_row + col0, w);
                    return;
                }
#pragma unroll
                for (int q = 0; q < kUnit / 8; ++q)
                    *reinterpret_cast<uint4*>(buf + staged(lane, q)) = make_uint4(w[4 * q], w[4 * q + 1], w[4 * q + 2], w[4 * q + 3]);
                __syncwarp();
                stage_out(buf, out_at, e, row0, col0, lane);
                __syncwarp();
            };
            const uint32_t tmem_rows = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
            const float nan = __uint_as_float(0x7fc00000u);  // what a wait that gave up leaves: never plausible numbers
            const uint16_t* const residual_row = residual + static_cast<int64_t>(row) * e.residual_stride;
            auto fetch = [&](int col0) {
                if (e.residual_piece == 32) {
                    if (live && col0 < e.n) load_row32(ahead, residual_row + col0);
                } else {
                    fetch_unit(ahead, residual_at, col0, e.n, e.residual_piece, lane);
                }
            };
            if (e.residual) fetch(tn * p.tile_n + turn * kUnit);
            // The first tile starts with a pass beyond the last column, which loads and stores nothing: it brings
            // the code below into the instruction cache while the first MMAs run.
#pragma unroll 1
            for (int j = t == pair ? -1 : 0, u = turn + kUnitWarps * j; u < units; ++j, u += kUnitWarps) {
                const int col0 = j < 0 ? e.n : tn * p.tile_n + u * kUnit;
                if (j == 0) {
                    if (ok) ok = mbar_wait(acc_full + 8 * acc, acc_phase, abort_flag, 5, limit);
                    ok = __all_sync(0xffffffffu, ok);
                    tc_fence_after();
                }
                uint64_t v[kUnit / 2];
                {
                    uint32_t bits[16];
                    if (ok && j >= 0) {
                        tmem_ld16(tmem_rows + acc * 256 + u * kUnit, bits);
                        tmem_wait_ld();
                    } else {
#pragma unroll
                        for (int i = 0; i < kUnit; ++i) bits[i] = __float_as_uint(nan);
                    }
#pragma unroll
                    for (int i = 0; i < kUnit / 2; ++i) v[i] = pack2(__uint_as_float(bits[2 * i]), __uint_as_float(bits[2 * i + 1]));
                }
                if (col0 >= e.n && j >= 0) continue;
                uint32_t old[kUnit / 2] = {};
                if (e.residual && j >= 0) {
                    if (e.residual_piece != 32) turn_unit(buf, ahead, lane);
#pragma unroll
                    for (int i = 0; i < kUnit / 2; ++i) old[i] = ahead[i];
                    if (u + kUnitWarps < units) fetch(col0 + kUnitWarps * kUnit);
                }
                finish(v, old, j < 0 ? 0 : j, col0);
            }
            if (units <= turn) {  // a tile with fewer units than warps: this one only hands the accumulator back
                if (ok) ok = mbar_wait(acc_full + 8 * acc, acc_phase, abort_flag, 5, limit);
                ok = __all_sync(0xffffffffu, ok);
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
constexpr int kSwapMaxStages = 8;
constexpr int kSwapCtlBytes = 16 * kSwapMaxStages + 64;

template <bool kFp8>
__global__ void __launch_bounds__(kSwapThreads) linear_swap_kernel(const __grid_constant__ LinearParams p) {
    extern __shared__ char smem_raw[];
    char* smem = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    const uint32_t step_bytes = kRowTile + static_cast<uint32_t>(p.tile_n) * kStepBytes;
    char* ctl = smem + p.stages * kSub * step_bytes;
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
    allow_next_kernel();
    if (warp == 1) {
        tmem_alloc(smem_u32(tmem_slot), p.tmem_cols);
        tmem_relinquish();
    }
    wait_for_kernels_before();
    tc_fence_before();
    const bool dead = __syncthreads_or(threadIdx.x == 0 && p.status && *reinterpret_cast<volatile int*>(p.status) != 0);
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    bool ok = !dead;

    const Epilogue& e = p.e;
    const int quarter = warp & 3;  // warps 2..5 cover the four quarters of the 128 lanes
    const int channel = row_w + lane * 4;
    float b[4] = {}, scale[4] = {};
    // The finished values of four consecutive channels of one token.
    auto finish = [&](float (&v)[4], int token, int first) {
        const int64_t row = row_x + token;
        if (kFp8) {
            const float xs = __ldg(e.x_scale + row * e.x_scale_step);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = v[i] * xs * scale[i];
        }
        uint64_t pairs[2] = {pack2(v[0] + b[0], v[1] + b[1]), pack2(v[2] + b[2], v[3] + b[3])};
        activate(pairs, e.act);
        unpack2(pairs[0], v[0], v[1]);
        unpack2(pairs[1], v[2], v[3]);
        if (e.gate) {
            const int64_t at = static_cast<int64_t>(static_cast<uint32_t>(row) / e.rows_per_gate) * e.gate_stride + first;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (first + i < e.n) v[i] *= load_any(e.gate, e.gate_type, at + i);
        }
        if (e.residual) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (first + i < e.n)
                    v[i] += load_any(e.residual, e.out_fp16 ? MINDIESD_FP16 : MINDIESD_BF16, row * e.residual_stride + first + i);
        }
        const uint32_t lo = pack_pair(v[0], v[1], e.out_fp16), hi = pack_pair(v[2], v[3], e.out_fp16);
        uint16_t* o = static_cast<uint16_t*>(e.out) + row * e.out_stride + first;
        if (e.out_piece >= 8) {  // n is a multiple of 4 then
            if (first < e.n) *reinterpret_cast<uint2*>(o) = make_uint2(lo, hi);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (first + i < e.n) o[i] = static_cast<uint16_t>((i < 2 ? lo : hi) >> ((i & 1) * 16));
        }
    };
    if (warp >= 2) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            b[i] = e.bias && channel + i < e.n ? load_any(e.bias, e.bias_type, channel + i) : 0.0f;
            scale[i] = kFp8 && channel + i < e.n ? __ldg(e.w_scale + static_cast<int64_t>(channel + i) * e.w_scale_step) : 0.0f;
        }
    }

    if (warp == 0) {
        if (ok && !p.test_withhold) {
            const bool one = elect_one();
            const uint32_t ring = smem_u32(smem);
            int stage = 0;
            uint32_t phase = 0;
            for (int ks = ks0; ks < ks1; ks += kSub) {
                ok = mbar_wait_warp(empty + 8 * stage, phase ^ 1, abort_flag, 6, limit);
                if (!ok) break;
                const int subs = min(kSub, ks1 - ks);
                if (one) {
                    mbar_arrive_expect_tx(full + 8 * stage, subs * step_bytes);
                    uint32_t dst = ring + stage * kSub * step_bytes;
                    for (int j = 0; j < subs; ++j, dst += step_bytes) {
                        tma_load_4d(dst, &p.tm_w, full + 8 * stage, (ks + j) * p.k_step_elems, row_w, 0, 0);
                        tma_load_4d(dst + kRowTile, &p.tm_x, full + 8 * stage, (ks + j) * p.k_step_elems, row_x, 0, 0);
                    }
                }
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
        if (ok) {
            const bool one = elect_one();
            const uint32_t ring = smem_u32(smem);
            int stage = 0;
            uint32_t phase = 0;
            for (int ks = ks0; ks < ks1; ks += kSub) {
                if (!mbar_wait_warp(full + 8 * stage, phase, abort_flag, 7, limit)) break;
                tc_fence_after();
                const uint32_t a = desc_lo(ring + stage * kSub * step_bytes, 16);
                const uint32_t b = desc_lo(ring + stage * kSub * step_bytes + kRowTile, 16);
                if (one) {
#pragma unroll
                    for (int j = 0; j < kSub; ++j) {
                        if (ks + j >= ks1) break;
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            umma_ss_lohi<kFp8>(tmem, a + j * (step_bytes >> 4) + 2 * i, b + j * (step_bytes >> 4) + 2 * i,
                                               kDescHiSbo1024, p.idesc, ks > ks0 || (j | i) != 0);
                    }
                    umma_commit(empty + 8 * stage);
                }
                __syncwarp();
                if (++stage == p.stages) {
                    stage = 0;
                    phase ^= 1;
                }
            }
            if (one) umma_commit(done);  // also after a wait that gave up: the MMAs that were issued must be over
            mbar_wait_drain(done, 0);
        }
    }

    const int tokens = min(p.tile_n, e.m - row_x);
    float* partial = reinterpret_cast<float*>(smem);  // [token][128]
    auto meet = [&] {
        if (p.split > 1) cluster_sync_all();
        else __syncthreads();
    };
    if (warp >= 2) {  // a lane takes four channels of one token
        const uint32_t mine = smem_u32(partial) + lane * 16;
        // The loop starts with a pass beyond the last channel, which loads and stores nothing: it brings the code
        // below into the instruction cache while the weights are on their way.
        int t = -1;
#pragma unroll 1
        do {
            float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            if (t >= 0) {  // every partial sum is on its way at once, and added in the order of the ranks
                float4 part[8];
#pragma unroll
                for (int r = 0; r < 8; ++r)
                    if (r < p.split) part[r] = cluster_load_f32x4(cluster_map(mine + t * 512, r));
#pragma unroll
                for (int r = 0; r < 8; ++r)
                    if (r < p.split) {
                        v[0] += part[r].x;
                        v[1] += part[r].y;
                        v[2] += part[r].z;
                        v[3] += part[r].w;
                    }
            }
            finish(v, t < 0 ? 0 : t, t < 0 ? e.n : channel);
            if (t >= 0) {
                t += p.split * 4;
                continue;
            }
            if (ok) ok = mbar_wait(done, 0, abort_flag, 8, limit);
            __syncwarp();
            ok = __syncthreads_and(ok && abort_flag[0] == 0);  // with warps 0 and 1: the ring is free
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < tokens; c += 16) {
                uint32_t r[16];
                if (ok) {
                    tmem_ld16(tmem + (static_cast<uint32_t>(quarter * 32) << 16) + c, r);
                    tmem_wait_ld();
                }
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    partial[(c + i) * 128 + quarter * 32 + lane] = ok ? __uint_as_float(r[i]) : __uint_as_float(0x7fc00000u);  // NaN
            }
            tc_fence_before();
            __syncwarp();
            meet();
            t = rank * 4 + quarter;
        } while (t < tokens);
    } else {
        __syncwarp();
        __syncthreads_and(ok && abort_flag[0] == 0);
        meet();
    }
    __syncwarp();
    if (p.split > 1) cluster_sync_all();  // the partials are read by the other blocks until here
    __syncthreads();
    if (warp == 1) tmem_dealloc(tmem, p.tmem_cols);
    if (threadIdx.x == 0) report(p, abort_flag);
}

// ---- host --------------------------------------------------------------------------------------------------

constexpr int kSms = 148;
constexpr int kMaxSmem = 227 * 1024;

// A launch configuration whose clusters span the x dimension, and whose start may overlap the kernel before it.
struct ClusterLaunch {
    cudaLaunchAttribute attr[2];
    cudaLaunchConfig_t cfg = {};
    ClusterLaunch(dim3 grid, int cluster, int threads, int smem, cudaStream_t stream) {
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = cluster;
        attr[0].val.clusterDim.y = 1;
        attr[0].val.clusterDim.z = 1;
        attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[1].val.programmaticStreamSerializationAllowed = 1;
        cfg.gridDim = grid;
        cfg.blockDim = dim3(threads, 1, 1);
        cfg.dynamicSmemBytes = smem;
        cfg.stream = stream;
        cfg.attrs = attr;
        cfg.numAttrs = 2;
    }
};

// Lets a kernel use all of an SM's shared memory, once per device (a call that set the limit to its own need could
// lower it under another thread's launch).
template <auto kKernel>
cudaError_t allow_all_shared_memory() {
    constexpr int kMaxDevices = 64;
    static std::atomic<bool> done[kMaxDevices];
    int dev = 0;
    cudaError_t err = cudaGetDevice(&dev);
    if (err != cudaSuccess || (dev < kMaxDevices && done[dev].load(std::memory_order_acquire))) return err;
    err = cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem);
    if (err == cudaSuccess && dev < kMaxDevices) done[dev].store(true, std::memory_order_release);
    return err;
}

template <auto kKernel>
cudaError_t launch_clusters(const LinearParams& p, dim3 grid, int cluster, int threads, int smem, cudaStream_t stream) {
    const cudaError_t err = allow_all_shared_memory<kKernel>();
    if (err != cudaSuccess) return err;
    ClusterLaunch launch(grid, cluster, threads, smem, stream);
    return cudaLaunchKernelEx(&launch.cfg, kKernel, p);
}

// k steps per ring stage of the pair kernel: two halve the barriers' round trips, one makes better use of the ring
// where two of a tile's steps do not divide it (512 x 4096 x 5120 bf16: 160 columns 22.4 us with one, 24.8 with two;
// 2048 x 5120 x 5120: 192 columns 75 and 79 us, 128 columns 94 and 86, 256 columns 89 and 85).
constexpr int pair_sub(int tile_n) { return tile_n <= 128 || tile_n == 256 ? 2 : 1; }

template <bool kFp8>
cudaError_t launch_pair(const LinearParams& p, cudaStream_t stream) {
    const int tiles = p.tiles_m * p.tiles_n;
    const dim3 grid(2 * (tiles < kSms / 2 ? tiles : kSms / 2));
    return pair_sub(p.tile_n) == 1
               ? launch_clusters<linear_pair_kernel<kFp8, 1>>(p, grid, 2, kPairThreads, kPairSmem, stream)
               : launch_clusters<linear_pair_kernel<kFp8, 2>>(p, grid, 2, kPairThreads, kPairSmem, stream);
}

// How a product is cut up.
struct Plan {
    bool swap;
    int tile_n;  // pair: columns, swap: tokens
    int stages;
    int split;   // swap: blocks of a cluster that share the k of a tile
    int band;    // pair
};

constexpr int swap_columns(int tile_n) { return tile_n <= 32 ? 32 : tile_n <= 64 ? 64 : 128; }
constexpr int swap_smem(int tile_n, int stages) { return stages * kSub * (kRowTile + tile_n * kStepBytes) + kSwapCtlBytes + 1024; }
constexpr int kSwapMaxTile = 128, kSwapMaxSplit = 8;

// Stages that let `per_sm` blocks of the swap kernel share an SM (1 KB of each goes to the system).  Blocks that fit
// by their shared memory also fit by their tensor memory (at most 2 x 128 columns of 512), so an allocation of
// one never waits for another block of its kind.
constexpr int swap_stages(int tile_n, int per_sm) {
    const int stages = (228 * 1024 / per_sm - 1024 - swap_smem(0, 0)) / (kSub * (kRowTile + tile_n * kStepBytes));
    return stages < kSwapMaxStages ? stages : kSwapMaxStages;
}
constexpr int pair_stages(int tile_n) {
    const int stages = kRingBytes / (pair_sub(tile_n) * (kRowTile + tile_n / 2 * kStepBytes));
    return stages < kPairMaxStages ? stages : kPairMaxStages;
}

// Row tiles of a band (tile_at).  All of w passes by once per band, so where w does not stay in L2 the band is as high
// as its rows of x leave room for (32760 x 5120 x 20480 bf16 under the power cap, w 210 MB: 4 tiles 5.66 ms, 8 tiles
// 5.29, 16 tiles 5.18); where it does, a low band keeps the tiles in flight close (32768 x 5120 x 5120 e4m3, w 26 MB:
// 4 tiles 694 us, 16 tiles 709).
constexpr int pair_band(int n, int k_steps) {
    const int64_t row_bytes = static_cast<int64_t>(k_steps) * kStepBytes;
    if (n * row_bytes <= (40 << 20)) return 4;
    const int64_t band = (44 << 20) / (256 * row_bytes);
    return band < 4 ? 4 : band > 16 ? 16 : static_cast<int>(band);
}

// Clusters of 1..8 blocks that the device holds at once with one and with two blocks per SM.  A cluster lies inside
// one group of SMs, so these are not 148 / size: measured 15 of eight blocks, not 18, and a 16th one is a second wave.
struct Residency {
    int clusters[2][kSwapMaxSplit + 1];
};
const Residency& residency() {
    constexpr int kMaxDevices = 64;
    static std::mutex mu;
    static Residency table[kMaxDevices];
    static bool known[kMaxDevices] = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) dev = 0;
    std::lock_guard<std::mutex> lock(mu);
    Residency& r = table[dev];
    if (!known[dev]) {
        allow_all_shared_memory<linear_swap_kernel<false>>();
        for (int per_sm = 1; per_sm <= 2; ++per_sm) {
            const int smem = swap_smem(16, swap_stages(16, per_sm));
            for (int size = 1; size <= kSwapMaxSplit; ++size) {
                ClusterLaunch launch(dim3(size), size, kSwapThreads, smem, nullptr);
                int n = 0;
                if (cudaOccupancyMaxActiveClusters(&n, linear_swap_kernel<false>, &launch.cfg) != cudaSuccess || n <= 0) {
                    cudaGetLastError();
                    n = kSms * per_sm / size;
                }
                r.clusters[per_sm - 1][size] = n;
            }
        }
        known[dev] = true;
    }
    return r;
}

// The plan with the smallest estimated time.  The estimates are a model of the two kernels (microseconds) whose
// constants were fitted to 8700 timings of 300 products (m 1..16000, k 64..20480, n 16..20480, both operand
// widths): the plan it picks is 1.8 % slower than the best measured one on average, on 300 other products too, and
// more than 10 % slower for one in twenty.  What it weighs, with both sides measured (bf16, k 5120, n 5120):
//   m 64:   swap, 3 blocks per tile 16.0 us, 8 blocks 23 us (clusters of a second wave); pair 21.3 us
//   m 256:  pair, 96 columns (54 tiles) 21.3 us, 256 columns (20 tiles) 32 us; swap 26.3 us
//   m 2048: pair, 192 columns (216 tiles, 2.92 waves) 75 us, 256 columns (160 tiles, 2.16 waves) 85 us
// (Two launches, the columns of the full waves and then the rest, gained at most 8 % and lost as often.)
Plan estimate_plan(int m, int n, int k_steps) {
    auto ceil_div = [](int64_t x, int64_t y) { return (x + y - 1) / y; };
    const double bytes = (static_cast<double>(m) + n) * k_steps * kStepBytes + 2.0 * m * n;
    // The larger of the two times, and a share of the smaller one that the other does not hide.
    auto overlap = [](double busy, double memory, double share) { return std::max(busy, memory) + share * std::min(busy, memory); };
    constexpr double kMemory = 5.38e6, kMemoryOfBlock = 60e3;  // bytes per microsecond: 5.38 TB/s, 60 GB/s for one block
    Plan best = {};
    double best_us = 1e300;
    for (int tile_n = 32; tile_n <= 256; tile_n += 32) {
        if (tile_n > ceil_div(n, 32) * 32) break;
        const int64_t tiles = ceil_div(m, 256) * ceil_div(n, tile_n);
        const double waves = static_cast<double>(ceil_div(tiles, kSms / 2));
        // A k step of a tile: its MMAs, the round trip of its barriers, or the pairs' loads from L2 at 22.8 TB/s.
        double step = std::max(0.199, 0.00117 * tile_n);
        step = std::max(step, static_cast<double>(std::min<int64_t>(tiles, kSms / 2)) * 2 * (kRowTile + tile_n * 64) / 22.8e6);
        const double units = static_cast<double>(ceil_div(tile_n / kUnit, kUnitWarps));
        const double us = 3.28 + overlap(waves * std::max(k_steps * step, units), bytes / kMemory, 0.127) + 0.236 * units + 1.16 * waves;
        if (us < best_us) {
            best_us = us;
            best = {false, tile_n, pair_stages(tile_n), 1, pair_band(n, k_steps)};
        }
    }
    const int64_t blocks_n = ceil_div(n, 128);
    int last = 0;
    for (int want = 16; want <= kSwapMaxTile; want += 16) {
        const int64_t parts = ceil_div(m, want);
        if (blocks_n > 65535 || (parts > 1 && blocks_n * parts > 2 * kSms * 2)) continue;  // (the grid; w read by many blocks)
        const int tile = static_cast<int>(ceil_div(ceil_div(m, parts), 16) * 16);  // even parts
        if (tile == last) continue;
        last = tile;
        for (int per_sm = 1; per_sm <= 2; ++per_sm) {
            const int stages = swap_stages(tile, per_sm);
            if (stages < 2) continue;
            for (int split = 1; split <= kSwapMaxSplit && (split == 1 || k_steps >= 2 * split); ++split) {
                const int64_t clusters = blocks_n * parts, room = residency().clusters[per_sm - 1][split];
                const double waves = static_cast<double>(ceil_div(clusters, room));
                const double active = static_cast<double>(std::min(clusters, room)) * split;
                double step = std::max(0.219, 0.0033 * tile) * (1 + 0.69 * (std::max(1.0, active / kSms) - 1));
                step = std::max(step, active * (kRowTile + tile * kStepBytes) / 9.6e6);
                const double reduce = 0.076 * std::min(tile, m) / split + (split > 1 ? 1.04 : 0.0);
                const double steps = static_cast<double>(ceil_div(ceil_div(k_steps, split), kSub) * kSub);
                const double us = 2.66 + overlap(waves * steps * step, bytes / std::min(kMemory, active * kMemoryOfBlock), 0.089) + reduce * waves + 1.23 * (waves - 1);
                if (us < best_us) {
                    best_us = us;
                    best = {true, tile, stages, split, 0};
                }
            }
        }
    }
    return best;
}

// The plan depends on the sizes alone, so the estimates (2 us of host time) are made once for each.
Plan choose_plan(int m, int n, int k_steps) {
    struct Entry {
        int m, n, k_steps;
        Plan plan;
    };
    constexpr int kEntries = 64;
    thread_local Entry cache[kEntries] = {};
    const unsigned h = (static_cast<unsigned>(m) * 0x9e3779b1u) ^ (static_cast<unsigned>(n) * 0x85ebca6bu) ^
                       (static_cast<unsigned>(k_steps) * 0xc2b2ae35u);
    Entry& c = cache[(h ^ (h >> 15)) % kEntries];
    if (c.m != m || c.n != n || c.k_steps != k_steps) c = {m, n, k_steps, estimate_plan(m, n, k_steps)};
    return c.plan;
}

// The plan that a test asks for; false where it is none that choose_plan could return for some sizes.
bool given_plan(const mindiesd_linear_cut& c, int m, int n, int k_steps, Plan& plan) {
    if (c.few_rows == 0) {
        if (c.tile < 32 || c.tile > 256 || c.tile % 32 != 0 || c.tile >= static_cast<int64_t>(n) + 32 || c.split != 1 || c.blocks_per_sm != 1) return false;
        plan = {false, c.tile, pair_stages(c.tile), 1, pair_band(n, k_steps)};
        return true;
    }
    if (c.few_rows != 1 || c.tile < 16 || c.tile > kSwapMaxTile || c.tile % 16 != 0 || c.tile >= static_cast<int64_t>(m) + 16) return false;
    if (c.split < 1 || c.split > kSwapMaxSplit || (c.split > 1 && k_steps < 2 * c.split)) return false;
    if (c.blocks_per_sm < 1 || c.blocks_per_sm > 2 || swap_stages(c.tile, c.blocks_per_sm) < 2) return false;
    plan = {true, c.tile, swap_stages(c.tile, c.blocks_per_sm), c.split, 0};
    return true;
}

template <bool kFp8>
cudaError_t launch_swap(const LinearParams& p, cudaStream_t stream) {
    const dim3 grid(p.split, (p.e.n + 127) / 128, (p.e.m + p.tile_n - 1) / p.tile_n);
    return launch_clusters<linear_swap_kernel<kFp8>>(p, grid, p.split, kSwapThreads, swap_smem(p.tile_n, p.stages), stream);
}

}  // namespace
}  // namespace sdb

using namespace sdb;

// cut: null, or how a test wants the product cut up.
static int linear_fwd(const mindiesd_linear_args* a, const mindiesd_linear_cut* cut, void* stream_) try {
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
    // The largest piece that every row starts on and holds a whole number of.
    auto piece_of = [&](const void* ptr, int64_t stride) {
        const uintptr_t bits = reinterpret_cast<uintptr_t>(ptr) | static_cast<uintptr_t>(stride) * 2 | static_cast<uintptr_t>(a->n) * 2;
        return bits % 32 == 0 ? 32 : bits % 16 == 0 ? 16 : bits % 8 == 0 ? 8 : 2;
    };
    e.out_piece = piece_of(a->out, e.out_stride);
    e.residual_piece = a->residual ? piece_of(a->residual, a->residual_stride) : 32;
    e.wide_gate = a->gate && aligned(a->gate, 16) && (a->gate_stride * dtype_bytes(a->gate_dtype)) % 16 == 0;
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
    Plan plan;
    if (!cut) plan = choose_plan(a->m, a->n, p.k_steps);
    else if (!given_plan(*cut, a->m, a->n, p.k_steps, plan)) return MINDIESD_E_VALUE;
    p.tile_n = plan.tile_n;
    p.split = plan.split;
    p.stages = plan.stages;
    if (plan.swap) {
        p.tmem_cols = swap_columns(p.tile_n);
        p.idesc = umma_idesc(fmt, 128, p.tile_n, false, false);
        if ((a->n + 127) / 128 > 65535 || (a->m + p.tile_n - 1) / p.tile_n > 65535) return MINDIESD_E_CAPACITY;
        if ((rc = encode_tile_map(&p.tm_w, a->weight, a->in_dtype, a->k, a->n, 1, 1, w_strides, 128))) return rc;
        if ((rc = encode_tile_map(&p.tm_x, a->x, a->in_dtype, a->k, a->m, 1, 1, x_strides, p.tile_n))) return rc;
        err = fp8 ? launch_swap<true>(p, stream) : launch_swap<false>(p, stream);
    } else {
        p.tiles_m = (a->m + 255) / 256;
        p.tiles_n = (a->n + p.tile_n - 1) / p.tile_n;
        if (static_cast<int64_t>(p.tiles_m) * p.tiles_n > 0x3fffffff) return MINDIESD_E_CAPACITY;
        p.band = plan.band;
        p.idesc = umma_idesc(fmt, 256, p.tile_n, false, false);
        if ((rc = encode_tile_map(&p.tm_x, a->x, a->in_dtype, a->k, a->m, 1, 1, x_strides, 128))) return rc;
        if ((rc = encode_tile_map(&p.tm_w, a->weight, a->in_dtype, a->k, a->n, 1, 1, w_strides, p.tile_n / 2))) return rc;
        err = fp8 ? launch_pair<true>(p, stream) : launch_pair<false>(p, stream);
    }
    if (err == cudaSuccess) return MINDIESD_OK;
    cudaGetLastError();  // the caller gets the error from here; the next call's check must not find it again
    return static_cast<int>(err);
} catch (...) {  // a lock that the system refused; nothing may cross this boundary
    return MINDIESD_E_DRIVER;
}

extern "C" int mindiesd_linear_fwd(const mindiesd_linear_args* a, void* stream) { return linear_fwd(a, nullptr, stream); }

extern "C" int mindiesd_linear_fwd_as(const mindiesd_linear_args* a, const mindiesd_linear_cut* cut, void* stream) {
    return cut ? linear_fwd(a, cut, stream) : MINDIESD_E_NULL;
}
