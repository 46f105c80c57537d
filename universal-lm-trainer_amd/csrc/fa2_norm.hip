// fa2_norm.hip -- RMS norm of token rows with the residual's addition in front
// of it, and the same with the normalised row in 8 bits.  (Gradient: fa2_norm_bwd.hip.)
//
//   h = residual + D(x)            (D: dropout, or nothing; h = x without a residual)
//   y = h * s * w,                 s = (mean(h^2) + eps)^-1/2
//   8 bits: scale = max(amax|y| / 448, 2^-126), q = e4m3(y / scale)
//
// h is rounded to the residual's type before the norm reads it, so that the
// gradient, which finds only that h, is the gradient of what was computed; sums
// and statistics are fp32.
//
// Bound by memory: one pass over the rows, each held in registers by the G lanes
// that share it (a wave up to 1024 columns, 256 or 1024 threads beyond), four
// elements a load.  32768 x 768, fp16 branch, fp32 residual: 49 us, 6.2 TB/s.
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

template <typename TX, typename TR, typename TY, int G, int NCH, bool STREAM>
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
        for (int c = 0; c < NCH; ++c) h[c] = load4<TX, STREAM>(x, (c * G + t) * 4, a.cols, vec);
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
            for (int c = 0; c < NCH; ++c) h[c] = load4<TR, STREAM>(r, (c * G + t) * 4, a.cols, vec) + h[c];
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

template <typename TX, typename TR, typename TY>
hipError_t fwd(const NormFwdArgs &a, hipStream_t st) {
    return by_cols(a.cols, [&](auto g, auto n) {
        constexpr int G = decltype(g)::value, RPB = (G > 256 ? G : 256) / G;
        const int64_t want = (a.rows + RPB - 1) / RPB, most = 1 << 20;   // 2^30 threads; more rows take turns
        const dim3 grid((unsigned)(want < most ? want : most)), block(G > 256 ? G : 256);
        if (a.stream)
            hipLaunchKernelGGL((norm_fwd_kernel<TX, TR, TY, G, decltype(n)::value, true>), grid, block, 0, st, a);
        else
            hipLaunchKernelGGL((norm_fwd_kernel<TX, TR, TY, G, decltype(n)::value, false>), grid, block, 0, st, a);
        return hipGetLastError();
    });
}

}  // namespace

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

}  // namespace fa2
