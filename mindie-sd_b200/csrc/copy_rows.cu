// Copies rows of bytes to rows of a padded stride, so that the tensor copies of the matrix product can fetch them.
//
// Bound by HBM: every byte is read and written once.  A warp takes 2 KB of a row, four 16-byte chunks per lane, all loads
// before the first store.  Where the source lies on less than 16 bytes a chunk is put together from narrower loads,
// which hit the lines that the first of them brought.
#include "ptx_sm100.cuh"
#include "row_io.cuh"

namespace sdb {
namespace {

constexpr int kWarps = 8;
constexpr int kChunks = 4;                   // of 16 bytes, per lane
constexpr int kSegment = 32 * kChunks * 16;  // bytes of a row per warp

template <int kBytes>
__global__ void __launch_bounds__(32 * kWarps) copy_rows_kernel(const mindiesd_copy_rows_args a, int64_t segments) {
    using Piece = typename Raw<kBytes>::type;
    constexpr int kPieces = 16 / kBytes;
    allow_next_kernel();
    wait_for_kernels_before();
    const int64_t unit = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
    const int64_t row = unit / segments;
    if (row >= a.rows) return;
    const int64_t first = (unit - row * segments) * kSegment + (threadIdx.x & 31) * 16;
    const char* src = static_cast<const char*>(a.src) + row * a.src_stride;
    char* dst = static_cast<char*>(a.dst) + row * a.dst_stride;
    union Chunk {
        Piece piece[kPieces];
        uint4 all;
        __device__ __forceinline__ Chunk() : all(make_uint4(0, 0, 0, 0)) {}
    } chunk[kChunks];
#pragma unroll
    for (int j = 0; j < kChunks; ++j)
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            const int64_t at = first + j * 512 + i * kBytes;
            if (at < a.row_bytes) chunk[j].piece[i] = __ldg(reinterpret_cast<const Piece*>(src + at));
        }
#pragma unroll
    for (int j = 0; j < kChunks; ++j) {
        const int64_t at = first + j * 512;
        if (at < a.row_bytes) *reinterpret_cast<uint4*>(dst + at) = chunk[j].all;
    }
}

template <int kBytes>
cudaError_t launch(const mindiesd_copy_rows_args& a, cudaStream_t stream) {
    const int64_t segments = (a.row_bytes + kSegment - 1) / kSegment;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>((a.rows * segments + kWarps - 1) / kWarps));
    cfg.blockDim = dim3(32 * kWarps);
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, copy_rows_kernel<kBytes>, a, segments);
}

}  // namespace
}  // namespace sdb

using namespace sdb;

extern "C" int mindiesd_copy_rows(const mindiesd_copy_rows_args* a, void* stream_) {
    if (!a || !a->src || !a->dst) return MINDIESD_E_NULL;
    if (a->rows <= 0 || a->row_bytes <= 0) return MINDIESD_E_SHAPE;
    if (a->rows > 0x7fffffff || a->row_bytes > 0x1ffffffffLL) return MINDIESD_E_CAPACITY;
    if ((a->rows * ((a->row_bytes + kSegment - 1) / kSegment) + kWarps - 1) / kWarps > 0x7fffffff) return MINDIESD_E_CAPACITY;
    const int64_t padded = (a->row_bytes + 15) / 16 * 16;
    if (a->src_stride < 0 || a->dst_stride < padded || a->dst_stride % 16 != 0) return MINDIESD_E_STRIDE;
    if (reinterpret_cast<uintptr_t>(a->dst) % 16 != 0) return MINDIESD_E_STRIDE;
    const uintptr_t s = reinterpret_cast<uintptr_t>(a->src), d = reinterpret_cast<uintptr_t>(a->dst);
    if (s < d + static_cast<uintptr_t>((a->rows - 1) * a->dst_stride + padded) && d < s + static_cast<uintptr_t>((a->rows - 1) * a->src_stride + a->row_bytes))
        return MINDIESD_E_VALUE;
    // The widest piece that every row starts on and that divides a row: no load passes a row's end.
    const uint64_t bits = s | static_cast<uint64_t>(a->src_stride) | static_cast<uint64_t>(a->row_bytes) | 16;
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    cudaError_t err;
    if (bits % 16 == 0) err = launch<16>(*a, stream);
    else if (bits % 8 == 0) err = launch<8>(*a, stream);
    else if (bits % 4 == 0) err = launch<4>(*a, stream);
    else if (bits % 2 == 0) err = launch<2>(*a, stream);
    else err = launch<1>(*a, stream);
    if (err == cudaSuccess) return MINDIESD_OK;
    cudaGetLastError();  // the caller gets the error from here; the next call's check must not find it again
    return static_cast<int>(err);
}
