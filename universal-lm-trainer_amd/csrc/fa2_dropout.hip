// fa2_dropout.hip -- dropout of token rows from a counter-based generator.
//
// y[r, c] = x[r, c] / (1 - p) where keep(seed, r, c), else 0; the product is
// fp32 and rounded once.  keep is the attention dropout's hash of the seed, the
// row and the column (fa2_device.h, head 0), so nothing but the seed is kept for
// the gradient, which is the same kernel on dy.
//
// One pass, each thread a piece of E elements of a row at a time (eight, one 16-byte
// load of fp16, where rows are made of such; else four, loaded by a type aligned to its
// elements only, the last piece of a row by element); a division finds its first row
// and column, later ones are found by adding the grid's stride in rows and columns.
// Bound by memory: 32768 x 768 in fp16 take 17 to 19 us, 5.4 to 5.8 TB/s (nontemporal
// loads or stores change nothing).
#include "fa2_token.h"

namespace fa2 {
namespace {

template <typename T, int E>
__global__ __launch_bounds__(256) void dropout_kernel(const DropoutArgs a) {
    const uint32_t nc = ((uint32_t)a.cols + E - 1) / E;          // pieces of a row
    const uint64_t step = (uint64_t)gridDim.x * 256;
    const uint64_t at = (uint64_t)blockIdx.x * 256 + threadIdx.x;
    int64_t row = (int64_t)(at / nc);
    uint32_t c = (uint32_t)(at - (uint64_t)row * nc);
    const int64_t srow = (int64_t)(step / nc);
    const uint32_t sc = (uint32_t)(step - (uint64_t)srow * nc);
    while (row < a.rows) {
        const T *x = static_cast<const T *>(a.x) + row * a.x_stride + (int64_t)c * E;
        T *y = static_cast<T *>(a.y) + row * a.cols + (int64_t)c * E;
        const uint32_t part = a.seed_part ^ dropout_row_term((int)row);
        const int col = (int)(c * E);
        if (E == 8) {
            typedef typename vec_of<T>::v8 v8;
            f8 v = __builtin_convertvector(*reinterpret_cast<const v8 *>(x), f8);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = drop(v[j], part, col + j, a.drop_thr, a.inv_keep);
            *reinterpret_cast<v8 *>(y) = __builtin_convertvector(v, v8);
        } else {
            f4 v = load4(x, 0, a.cols - col, false);
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = drop(v[j], part, col + j, a.drop_thr, a.inv_keep);
            store4(y, 0, a.cols - col, false, v);
        }
        row += srow;
        c += sc;
        if (c >= nc) {
            c -= nc;
            ++row;
        }
    }
}

template <typename T>
hipError_t run(const DropoutArgs &a, hipStream_t st) {
    const uint64_t pieces = (uint64_t)a.rows * (a.vec ? a.cols / 8 : (a.cols + 3) / 4);
    const uint64_t want = (pieces + 255) / 256;
    const dim3 grid((unsigned)(want < 8192 ? want : 8192)), block(256);
    if (a.vec)
        hipLaunchKernelGGL((dropout_kernel<T, 8>), grid, block, 0, st, a);
    else
        hipLaunchKernelGGL((dropout_kernel<T, 4>), grid, block, 0, st, a);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_dropout(const DropoutArgs &a, int type, hipStream_t st) {
    if (type == FA2_F16) return run<_Float16>(a, st);
    if (type == FA2_BF16) return run<__bf16>(a, st);
    return run<float>(a, st);
}

}  // namespace fa2
