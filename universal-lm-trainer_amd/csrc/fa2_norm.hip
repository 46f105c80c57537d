// fa2_norm.hip -- RMS norm of token rows with the residual's addition in front
// of it, its gradient, and a forward that leaves the normalised row in 8 bits.
//
//   h = residual + D(x)            (D: dropout, or nothing; h = x without a residual)
//   y = h * s * w,                 s = (mean(h^2) + eps)^-1/2
//   8 bits: scale = max(amax|y| / 448, 2^-126), q = e4m3(y / scale)
//   backward, with g = dy * w and n = h * s:
//     total = s * (g - n * mean(g * n)) + dh;  dresidual = total,  dx = D'(total)
//     dw = sum over rows of dy * n
//
// h is rounded to the residual's type before the norm reads it, so that the
// gradient, which finds only that h, is the gradient of what was computed; sums
// and statistics are fp32.
//
// Bound by memory: one pass over the rows, each held in registers by the G lanes
// that share it (a wave up to 1024 columns, 256 or 1024 threads beyond), four
// elements a load.  The backward's workgroups run over many rows each and keep
// their part of dw in registers; the parts are summed in a second kernel in a
// fixed order, so that results do not change from run to run.
#include <type_traits>

#include "fa2_token.h"

namespace fa2 {
namespace {

struct Fp8 {};   // output tag: e4m3 with one scale a row

constexpr float FP8_MAX = 448.f;
constexpr float FP8_MIN_SCALE = 1.17549435e-38f;   // 2^-126: its reciprocal is finite, and a row of zeros divides by it

__device__ __forceinline__ void store_fp8(uint8_t *row, int col, int cols, bool vec, f4 v) {
    int q = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false);
    q = __builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], q, true);
    typedef int any_int __attribute__((aligned(1)));
    if (vec) {
        if (col < cols) *reinterpret_cast<int *>(row + col) = q;
    } else if (col + 4 <= cols) {
        *reinterpret_cast<any_int *>(row + col) = q;
    } else {
#pragma unroll
        for (int j = 0; j < 3; ++j)
            if (col + j < cols) row[col + j] = (uint8_t)(q >> (8 * j));
    }
}

template <typename TY>
struct out_bytes {
    typedef TY type;
};
template <>
struct out_bytes<Fp8> {
    typedef uint8_t type;
};

template <typename TX, typename TR, typename TY, int G, int NCH>
__global__ __launch_bounds__(G > 256 ? G : 256) void norm_fwd_kernel(const NormFwdArgs a) {
    constexpr bool FP8 = __is_same(TY, Fp8);
    constexpr int RPB = (G > 256 ? G : 256) / G;   // rows a workgroup
    __shared__ float red[G > 64 ? G / 64 : 1];
    const int t = threadIdx.x % G;
    const bool vec = a.vec;
    for (int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / G; row < a.rows; row += (int64_t)gridDim.x * RPB) {
        const TX *x = static_cast<const TX *>(a.x) + row * a.x_stride;
        f4 h[NCH], w[NCH];
#pragma unroll
        for (int c = 0; c < NCH; ++c) h[c] = load4(x, (c * G + t) * 4, a.cols, vec);
        // 8 bits: mostly few rows, where the weights' latency counts.  (Loaded here for the others too, 138 -> 141 us forward
        // and backward at 32768 x 768.)
        if (FP8) {
#pragma unroll
            for (int c = 0; c < NCH; ++c) w[c] = load4_typed(a.w, a.w_type, (c * G + t) * 4, a.cols, vec);
        }
        if (a.drop_thr) {
            const uint32_t part = a.seed_part ^ dropout_row_term((int)row);
#pragma unroll
            for (int c = 0; c < NCH; ++c)
#pragma unroll
                for (int j = 0; j < 4; ++j) h[c][j] = drop(h[c][j], part, (c * G + t) * 4 + j, a.drop_thr, a.inv_keep);
        }
        if (a.res) {
#pragma clang fp contract(off)
            const TR *r = static_cast<const TR *>(a.res) + row * a.res_stride;
#pragma unroll
            for (int c = 0; c < NCH; ++c) h[c] = load4(r, (c * G + t) * 4, a.cols, vec) + h[c];
        }
        if (a.h) {
            TR *ho = static_cast<TR *>(a.h) + row * a.cols;
#pragma unroll
            for (int c = 0; c < NCH; ++c) {
                store4(ho, (c * G + t) * 4, a.cols, vec, h[c]);
                // what the stream holds is what is normalised
                h[c] = __builtin_convertvector(__builtin_convertvector(h[c], typename vec_of<TR>::v4), f4);
            }
        }
        if (!FP8) {
#pragma unroll
            for (int c = 0; c < NCH; ++c) w[c] = load4_typed(a.w, a.w_type, (c * G + t) * 4, a.cols, vec);
        }
        float ss = 0.f;
#pragma unroll
        for (int c = 0; c < NCH; ++c)
#pragma unroll
            for (int j = 0; j < 4; ++j) ss += h[c][j] * h[c][j];
        ss = row_reduce<G, false>(ss, red);
        const float s = 1.f / sqrtf(ss / (float)a.cols + a.eps);
        if (a.rstd && t == 0) a.rstd[row] = s;
        float amax = 0.f;
#pragma unroll
        for (int c = 0; c < NCH; ++c)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                h[c][j] = h[c][j] * s * w[c][j];
                if (FP8 && (c * G + t) * 4 + j < a.cols) {   // the zeros past the row's end times inf are no values
                    const float v = fabsf(h[c][j]);
                    amax = (v > amax || v != v) ? v : amax;
                }
            }
        if constexpr (FP8) {
            amax = row_reduce<G, true>(amax, red);
            float scale = amax / FP8_MAX;
            scale = scale < FP8_MIN_SCALE ? FP8_MIN_SCALE : scale;
            if (t == 0) a.scale[row] = scale;
            // A product by the reciprocal: within 2^-23 of the quotient, which moves a value only where it lies that
            // near the middle of two e4m3 steps.
            const float inv = 1.f / scale;
            uint8_t *y = static_cast<uint8_t *>(a.y) + row * a.cols;
#pragma unroll
            for (int c = 0; c < NCH; ++c) store_fp8(y, (c * G + t) * 4, a.cols, vec, h[c] * inv);
        } else {
            TY *y = static_cast<TY *>(a.y) + row * a.cols;
#pragma unroll
            for (int c = 0; c < NCH; ++c) store4(y, (c * G + t) * 4, a.cols, vec, h[c]);
        }
    }
}

template <typename TX, typename TR, typename TY, int G, int NCH>
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
            dy[c] = load4(dyr, (c * G + t) * 4, a.cols, vec);
            n[c] = load4(hr, (c * G + t) * 4, a.cols, vec);
        }
        if (a.dh) {
            const TR *dhr = static_cast<const TR *>(a.dh) + row * a.dh_stride;
#pragma unroll
            for (int c = 0; c < NCH; ++c) dh[c] = load4(dhr, (c * G + t) * 4, a.cols, vec);
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

// Calls f(G, NCH) with the lanes a row takes and the four-element pieces a lane.
template <typename F>
hipError_t by_cols(int cols, F f) {
#define FA2_COLS(g, n) if (cols <= 4 * (g) * (n)) return f(std::integral_constant<int, g>(), std::integral_constant<int, n>())
    FA2_COLS(64, 1);
    FA2_COLS(64, 2);
    FA2_COLS(64, 3);
    FA2_COLS(64, 4);
    FA2_COLS(256, 2);
    FA2_COLS(256, 3);
    FA2_COLS(256, 4);
    FA2_COLS(1024, 2);
#undef FA2_COLS
    return hipErrorInvalidValue;
}

template <typename TX, typename TR, typename TY>
hipError_t fwd(const NormFwdArgs &a, hipStream_t st) {
    return by_cols(a.cols, [&](auto g, auto n) {
        constexpr int G = decltype(g)::value, RPB = (G > 256 ? G : 256) / G;
        const int64_t want = (a.rows + RPB - 1) / RPB, most = 1 << 20;   // 2^30 threads; more rows take turns
        hipLaunchKernelGGL((norm_fwd_kernel<TX, TR, TY, G, decltype(n)::value>), dim3((unsigned)(want < most ? want : most)),
                           dim3(G > 256 ? G : 256), 0, st, a);
        return hipGetLastError();
    });
}

template <typename TX, typename TR, typename TY>
hipError_t bwd(const NormBwdArgs &a, hipStream_t st) {
    const hipError_t e = a.blocks == 0 ? hipSuccess : by_cols(a.cols, [&](auto g, auto n) {   // no rows: dw = 0
        constexpr int G = decltype(g)::value;
        hipLaunchKernelGGL((norm_bwd_kernel<TX, TR, TY, G, decltype(n)::value>), dim3((unsigned)a.blocks),
                           dim3(G > 256 ? G : 256), 0, st, a);
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

// x_type, res_type (= x_type or fp32), y_type (x_type; any where x is fp32; fp8).
hipError_t launch_norm_fwd(const NormFwdArgs &a, int x_type, int res_type, int y_type, hipStream_t st) {
    if (x_type == FA2_F16) {
        if (res_type == FA2_F16) return y_type == FA2_E4M3 ? fwd<_Float16, _Float16, Fp8>(a, st) : fwd<_Float16, _Float16, _Float16>(a, st);
        return y_type == FA2_E4M3 ? fwd<_Float16, float, Fp8>(a, st) : fwd<_Float16, float, _Float16>(a, st);
    }
    if (x_type == FA2_BF16) {
        if (res_type == FA2_BF16) return y_type == FA2_E4M3 ? fwd<__bf16, __bf16, Fp8>(a, st) : fwd<__bf16, __bf16, __bf16>(a, st);
        return y_type == FA2_E4M3 ? fwd<__bf16, float, Fp8>(a, st) : fwd<__bf16, float, __bf16>(a, st);
    }
    switch (y_type) {
        case FA2_F16: return fwd<float, float, _Float16>(a, st);
        case FA2_BF16: return fwd<float, float, __bf16>(a, st);
        case FA2_E4M3: return fwd<float, float, Fp8>(a, st);
        default: return fwd<float, float, float>(a, st);
    }
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
