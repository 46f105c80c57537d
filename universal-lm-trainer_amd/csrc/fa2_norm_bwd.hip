// fa2_norm_bwd.hip -- gradient of fa2_norm.hip: with g = dy * w, n = h * s,
//
//   total = s * (g - n * mean(g * n)) + dh;  dresidual = total,  dx = D'(total)
//   dw = sum over rows of dy * n
//
// where s is the forward's statistic and D' its dropout (formed again from the seed).
//
// Bound by memory, as the forward.  A workgroup runs over many rows and keeps its part
// of dw in registers; the parts are summed in a second kernel in a fixed order, so that
// results do not change from run to run.  32768 x 768, fp16 branch, fp32 residual: 69
// us, 5.8 TB/s, and 4 us for the parts.
#include "fa2_token.h"

namespace fa2 {
namespace {

template <typename TX, typename TR, typename TY, int G, int NCH, bool STREAM>
__global__ __launch_bounds__(G > 256 ? G : 256) void norm_bwd_kernel(const NormBwdArgs a) {
    constexpr int BLOCK = G > 256 ? G : 256, RPB = BLOCK / G;
    __shared__ float red[G > 64 ? G / 64 : 1];
    __shared__ f4 sum[RPB > 1 ? BLOCK : 1];
    const int t = threadIdx.x % G, sub = threadIdx.x / G;
    const bool vec = a.vec;
    f4 w[NCH], dw[NCH];
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
        w[c] = load4_typed(a.w, a.w_type, (c * G + t) * 4, a.cols, vec);
        dw[c] = f4{0.f, 0.f, 0.f, 0.f};
    }
    const float inv_cols = 1.f / (float)a.cols;
    for (int64_t row = (int64_t)blockIdx.x * RPB + sub; row < a.rows; row += (int64_t)gridDim.x * RPB) {
        const TY *dyr = static_cast<const TY *>(a.dy) + row * a.dy_stride;
        const TR *hr = static_cast<const TR *>(a.h) + row * a.h_stride;
        f4 dy[NCH], n[NCH], dh[NCH];
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            dy[c] = load4<TY, STREAM>(dyr, (c * G + t) * 4, a.cols, vec);
            n[c] = load4<TR, STREAM>(hr, (c * G + t) * 4, a.cols, vec);
        }
        if (a.dh) {
            const TR *dhr = static_cast<const TR *>(a.dh) + row * a.dh_stride;
#pragma unroll
            for (int c = 0; c < NCH; ++c) dh[c] = load4<TR, STREAM>(dhr, (c * G + t) * 4, a.cols, vec);
        } else {
#pragma unroll
            for (int c = 0; c < NCH; ++c) dh[c] = f4{0.f, 0.f, 0.f, 0.f};
        }
        const float s = a.rstd[row];
        float dot = 0.f;
#pragma unroll
        for (int c = 0; c < NCH; ++c)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                n[c][j] *= s;
                dw[c][j] += dy[c][j] * n[c][j];
                dy[c][j] *= w[c][j];
                dot += dy[c][j] * n[c][j];
            }
        dot = row_reduce<G, false>(dot, red) * inv_cols;
#pragma unroll
        for (int c = 0; c < NCH; ++c)
#pragma unroll
            for (int j = 0; j < 4; ++j) dh[c][j] += s * (dy[c][j] - n[c][j] * dot);
        if (a.dres) {
            TR *o = static_cast<TR *>(a.dres) + row * a.cols;
#pragma unroll
            for (int c = 0; c < NCH; ++c) store4(o, (c * G + t) * 4, a.cols, vec, dh[c]);
        }
        if (a.dx) {
            if (a.drop_thr) {
                const uint32_t part = a.seed_part ^ dropout_row_term((int)row);
#pragma unroll
                for (int c = 0; c < NCH; ++c)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        dh[c][j] = drop(dh[c][j], part, (c * G + t) * 4 + j, a.drop_thr, a.inv_keep);
            }
            TX *o = static_cast<TX *>(a.dx) + row * a.cols;
#pragma unroll
            for (int c = 0; c < NCH; ++c) store4(o, (c * G + t) * 4, a.cols, vec, dh[c]);
        }
    }
    if (!a.dw) return;
    float *part = a.part + (int64_t)blockIdx.x * a.cols;
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
        f4 v = dw[c];
        if (RPB > 1) {   // the workgroup's rows side by side: summed in their order
            __syncthreads();
            sum[threadIdx.x] = v;
            __syncthreads();
            if (sub > 0) continue;
#pragma unroll
            for (int i = 1; i < RPB; ++i) v += sum[i * G + t];
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if ((c * G + t) * 4 + j < a.cols) part[(c * G + t) * 4 + j] = v[j];
    }
}

// dw[c] = sum over the blocks of their parts: 16 columns a workgroup, whose 64 groups
// of 16 threads take every 64th block and are added in a fixed order.  (64 columns a
// workgroup of four waves, each adding a quarter of the blocks: 34 us at 768 columns.)
__global__ __launch_bounds__(1024) void norm_dw_kernel(const float *part, int blocks, int cols, void *dw, int type) {
    __shared__ float s[64][17];
    const int k = threadIdx.x & 15, g = threadIdx.x >> 4, c = blockIdx.x * 16 + k;
    float v = 0.f;
    if (c < cols)
        for (int b = g; b < blocks; b += 64) v += part[(int64_t)b * cols + c];
    s[g][k] = v;
    __syncthreads();
    // wave w adds columns w: lane = group
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    v = s[lane][w];
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o);
    if (lane == 0 && blockIdx.x * 16 + w < cols) store1_typed(dw, type, blockIdx.x * 16 + w, v);
}

template <typename TX, typename TR, typename TY>
hipError_t bwd(const NormBwdArgs &a, hipStream_t st) {
    const hipError_t e = a.blocks == 0 ? hipSuccess : by_cols(a.cols, [&](auto g, auto n) {   // no rows: dw = 0
        constexpr int G = decltype(g)::value;
        const dim3 grid((unsigned)a.blocks), block(G > 256 ? G : 256);
        if (a.stream)
            hipLaunchKernelGGL((norm_bwd_kernel<TX, TR, TY, G, decltype(n)::value, true>), grid, block, 0, st, a);
        else
            hipLaunchKernelGGL((norm_bwd_kernel<TX, TR, TY, G, decltype(n)::value, false>), grid, block, 0, st, a);
        return hipGetLastError();
    });
    if (e != hipSuccess || !a.dw) return e;
    hipLaunchKernelGGL(norm_dw_kernel, dim3((unsigned)((a.cols + 15) / 16)), dim3(1024), 0, st, a.part, a.blocks, a.cols,
                       a.dw, a.dw_type);
    return hipGetLastError();
}

}  // namespace

// Two workgroups of 256 threads a compute unit, no more than there are rows for.
int norm_bwd_blocks(int64_t rows, int cols) {
    const int rpb = cols <= 1024 ? 4 : 1;
    const int64_t want = (rows + rpb - 1) / rpb, most = cols <= 4096 ? 512 : 256;
    return (int)(want < most ? want : most);
}

hipError_t launch_norm_bwd(const NormBwdArgs &a, int x_type, int h_type, int y_type, hipStream_t st) {
    if (x_type == FA2_F16) return h_type == FA2_F16 ? bwd<_Float16, _Float16, _Float16>(a, st) : bwd<_Float16, float, _Float16>(a, st);
    if (x_type == FA2_BF16) return h_type == FA2_BF16 ? bwd<__bf16, __bf16, __bf16>(a, st) : bwd<__bf16, float, __bf16>(a, st);
    switch (y_type) {
        case FA2_F16: return bwd<float, float, _Float16>(a, st);
        case FA2_BF16: return bwd<float, float, __bf16>(a, st);
        default: return bwd<float, float, float>(a, st);
    }
}

}  // namespace fa2
