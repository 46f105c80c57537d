// fa2_xent.hip -- the language model head with its softmax cross entropy:
// loss and gradients from the hidden states, without the [tokens, vocabulary]
// logits ever being kept.
//
//   z = x W^T,  lse_i = log sum_v exp z_iv,  loss_i = lse_i - z_(i, t_i)
//   G_iv = c_i (exp(z_iv - lse_i) - [v = t_i]);   dx = G W,  dW = G^T x
//
// Forward: one product whose tiles end in a running maximum and sum of each
// token's row; each slice of the vocabulary leaves one pair a token, which a
// second kernel joins.  Backward, for one piece of the vocabulary after another:
// the piece's logits again, turned into P = factor * G and rounded to the
// operands' type in a scratch of [tokens, piece]; then dW of the piece's rows,
// which is complete, and the piece's share of dx, summed in fp32.
//
// Tokens that do not count are taken out first (packed rows), so that no product
// works on them and nothing in their states, inf and NaN included, reaches a result.
//
// Rounding P to 16 bits (its relative error is at most half a step, and the
// errors of a sum's many terms are independent) keeps both gradient products on
// the matrix units; the gradients themselves are rounded to the same type.  P is
// scaled so that its largest possible value is 2^15: in fp16 probabilities down
// to 2^-29 stay normal numbers.
#include "fa2_token.h"

namespace fa2 {
namespace {

constexpr float P_SCALE = 32768.f;

typedef unsigned int u4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ f16x mfma(h8 a, h8 b, f16x c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f16x mfma(b8 a, b8 b, f16x c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }

// ---------------------------------------------------------------------------
// Packing
// ---------------------------------------------------------------------------

// One workgroup: positions of the tokens that count, in order.
__global__ __launch_bounds__(1024) void xent_scan_kernel(const XentArgs a) {
    __shared__ int wave_sum[16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int before = 0;   // tokens that count in earlier rounds
    for (int64_t r0 = 0; r0 < a.rows; r0 += 1024) {
        const int64_t i = r0 + threadIdx.x;
        const int64_t t = i < a.rows ? a.target[i] : a.ignore;
        const bool in = i < a.rows && t != a.ignore;
        const uint64_t m = __ballot(in);
        if (lane == 0) wave_sum[wave] = __popcll(m);
        __syncthreads();
        int mine = before, all = before;
#pragma unroll
        for (int w = 0; w < 16; ++w) {
            mine += w < wave ? wave_sum[w] : 0;
            all += wave_sum[w];
        }
        mine += __popcll(m & ((1ull << lane) - 1));
        if (i < a.rows) a.pos[i] = in ? mine : -1;
        if (in) {
            a.rowmap[mine] = (int)i;
            a.tgt[mine] = t >= 0 && t < a.V ? (int)t : -1;
        }
        before = all;
        __syncthreads();
    }
    if (threadIdx.x == 0) a.count[0] = before;
    for (int j = before + threadIdx.x; j < a.rows_pad; j += 1024) {
        a.rowmap[j] = -1;
        a.tgt[j] = -1;
    }
}

// Packed copy of the hidden states, one wave a row; zeros behind the last token
// and the last column.
template <typename T>
__global__ __launch_bounds__(256) void xent_pack_kernel(const XentArgs a) {
    const int lane = threadIdx.x & 63;
    const int j = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (j >= a.rows_pad) return;
    const int r = a.rowmap[j];
    T *o = static_cast<T *>(a.xc) + (int64_t)j * a.dp;
    const T *x = static_cast<const T *>(a.x) + (int64_t)r * a.x_stride;
    const bool vec = a.x_stride % 8 == 0 && (reinterpret_cast<uintptr_t>(a.x) & 15) == 0;
    typedef typename vec_of<T>::v8 v8;
    for (int c = lane * 8; c < a.dp; c += 512) {
        v8 v = {};
        if (r >= 0) {
            if (vec && c + 8 <= a.d) {
                v = *reinterpret_cast<const v8 *>(x + c);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (c + e < a.d) v[e] = x[c + e];
            }
        }
        *reinterpret_cast<v8 *>(o + c) = v;
    }
}

// Copy of the weight with rows of dp elements, for hidden sizes or strides that
// the tiles' 16-byte loads do not take.
template <typename T>
__global__ __launch_bounds__(256) void xent_pad_weight_kernel(const T *w, int64_t stride, T *out, int V, int d, int dp) {
    for (int64_t r = blockIdx.x; r < V; r += gridDim.x)
        for (int c = threadIdx.x; c < dp; c += 256) out[r * dp + c] = c < d ? w[r * stride + c] : (T)0.f;
}

// ---------------------------------------------------------------------------
// A 128 x 128 tile of a product, D[m, n] = sum_k A[m, k] B[n, k], by four waves
// of 64 x 64.  ROWS operands are stored [m][k], the others [k][m].  K is a
// multiple of 32; rows (k rows of the others) at or past the given limit are
// read from the last one, columns past the limit of the others likewise.
// ---------------------------------------------------------------------------
constexpr int TM = 128, TN = 128, TK = 32, TLD = TK + 8;

template <typename T>
struct Operand {
    const T *p;
    int64_t ld;
    int first, limit;      // ROWS: first row of the tile, rows; else first column, columns (a multiple of 8)
    int klimit;            // not ROWS: k rows
};

template <typename T, bool ROWS>
__device__ __forceinline__ void stage(const Operand<T> &o, int k0, T (*s)[TLD]) {
    typedef typename vec_of<T>::v8 v8;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int id = threadIdx.x + 256 * i;
        if (ROWS) {
            const int r = id >> 2, c = (id & 3) * 8;
            const int64_t row = min(o.first + r, o.limit - 1);
            *reinterpret_cast<v8 *>(&s[r][c]) = *reinterpret_cast<const v8 *>(o.p + row * o.ld + k0 + c);
        } else {
            const int k = id >> 4, c = (id & 15) * 8;
            const int64_t row = min(k0 + k, o.klimit - 1);
            const v8 v = *reinterpret_cast<const v8 *>(o.p + row * o.ld + min(o.first + c, o.limit - 8));
#pragma unroll
            for (int e = 0; e < 8; ++e) s[c + e][k] = v[e];
        }
    }
}

template <typename T>
struct TileMem {
    T a[TM][TLD], b[TN][TLD];
};

template <typename T, bool AROWS, bool BROWS>
__device__ __forceinline__ void product_tile(const Operand<T> &A, const Operand<T> &B, int kbeg, int kend, TileMem<T> &s,
                                             f16x acc[2][2]) {
    typedef typename vec_of<T>::v8 v8;
    const int lane = threadIdx.x & 63, c = lane & 31, g2 = lane >> 5;
    const int wm = (threadIdx.x >> 6 & 1) * 64, wn = (threadIdx.x >> 7) * 64;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[i][j] = zero16();
    for (int k0 = kbeg; k0 < kend; k0 += TK) {
        __syncthreads();
        stage<T, AROWS>(A, k0, s.a);
        stage<T, BROWS>(B, k0, s.b);
        __syncthreads();
#pragma unroll
        for (int ks = 0; ks < TK; ks += 16) {
            v8 fa[2], fb[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                fa[i] = *reinterpret_cast<const v8 *>(&s.a[wm + 32 * i + c][ks + 8 * g2]);
                fb[i] = *reinterpret_cast<const v8 *>(&s.b[wn + 32 * i + c][ks + 8 * g2]);
            }
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) acc[i][j] = mfma(fa[i], fb[j], acc[i][j]);
        }
    }
}

// Element (i, j, r) of a wave's accumulators: row m0 + 8 (r / 4) + 4 g2 + r % 4 of
// the tile's M side, column c of its N side.
__device__ __forceinline__ int acc_row(int r, int g2) { return 8 * (r >> 2) + 4 * g2 + (r & 3); }

// ---------------------------------------------------------------------------
// Forward
// ---------------------------------------------------------------------------

__device__ __forceinline__ void join_max_sum(float &m, float &l, float m2, float l2) {
    const float n = fmaxf(m, m2);
    const float base = n == -INFINITY ? 0.f : n;
    l = l * __expf(m - base) + l2 * __expf(m2 - base);
    m = n;
}

// Maximum and sum of exp of each packed row over a slice of the vocabulary.  The
// M side are vocabulary rows, the N side tokens: a lane holds one token's logits.
template <typename T>
__global__ __launch_bounds__(256) void xent_stats_kernel(const XentArgs a) {
    __shared__ TileMem<T> s;
    __shared__ float sm[2][TN], sl[2][TN];
    const int nr = a.rows_pad / TN;
    const int rb = blockIdx.x % nr, split = blockIdx.x / nr;
    if (rb * TN >= a.count[0]) return;
    const int tiles = (a.V + TM - 1) / TM;
    const int t0 = (int)((int64_t)tiles * split / a.splits), t1 = (int)((int64_t)tiles * (split + 1) / a.splits);
    const int lane = threadIdx.x & 63, c = lane & 31, g2 = lane >> 5;
    const int wmi = threadIdx.x >> 6 & 1, wn = (threadIdx.x >> 7) * 64;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    const Operand<T> B = {static_cast<const T *>(a.xc), a.dp, rb * TN, a.rows_pad, 0};
    for (int t = t0; t < t1; ++t) {
        const Operand<T> A = {static_cast<const T *>(a.w), a.w_stride, t * TM, a.V, 0};
        f16x acc[2][2];
        product_tile<T, true, true>(A, B, 0, a.dp, s, acc);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            float top = m[j];
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    if (t * TM + wmi * 64 + 32 * i + acc_row(r, g2) >= a.V) acc[i][j][r] = -INFINITY;
                    top = fmaxf(top, acc[i][j][r]);
                }
            const float base = top == -INFINITY ? 0.f : top;
            l[j] *= __expf(m[j] - base);
            m[j] = top;
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int r = 0; r < 16; ++r) l[j] += __expf(acc[i][j][r] - base);
        }
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        join_max_sum(m[j], l[j], __shfl_xor(m[j], 32), __shfl_xor(l[j], 32));
        if (g2 == 0) {
            sm[wmi][wn + 32 * j + c] = m[j];
            sl[wmi][wn + 32 * j + c] = l[j];
        }
    }
    __syncthreads();
    if (threadIdx.x < TN) {
        float mm = sm[0][threadIdx.x], ll = sl[0][threadIdx.x];
        join_max_sum(mm, ll, sm[1][threadIdx.x], sl[1][threadIdx.x]);
        f2 *o = reinterpret_cast<f2 *>(a.part) + (int64_t)split * a.rows_pad + rb * TN + threadIdx.x;
        *o = f2{mm, ll};
    }
}

// One wave a packed row: joins the slices, and the target's logit as a product of
// its own.
template <typename T>
__global__ __launch_bounds__(256) void xent_join_kernel(const XentArgs a) {
    const int lane = threadIdx.x & 63;
    const int j = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (j >= a.count[0]) return;
    float m = -INFINITY, l = 0.f;
    for (int s = lane; s < a.splits; s += 64) {
        const f2 p = *(reinterpret_cast<const f2 *>(a.part) + (int64_t)s * a.rows_pad + j);
        join_max_sum(m, l, p[0], p[1]);
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) join_max_sum(m, l, __shfl_xor(m, o), __shfl_xor(l, o));
    const float lse = m + __logf(l);
    const int t = a.tgt[j];
    float z = 0.f;
    if (t >= 0) {
        const T *x = static_cast<const T *>(a.xc) + (int64_t)j * a.dp;
        const T *w = static_cast<const T *>(a.w) + (int64_t)t * a.w_stride;
        typedef typename vec_of<T>::v8 v8;
        for (int c = lane * 8; c < a.dp; c += 512) {
            const f8 xv = __builtin_convertvector(*reinterpret_cast<const v8 *>(x + c), f8);
            const f8 wv = __builtin_convertvector(*reinterpret_cast<const v8 *>(w + c), f8);
#pragma unroll
            for (int e = 0; e < 8; ++e) z += xv[e] * wv[e];
        }
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) z += __shfl_xor(z, o);
    }
    if (lane == 0) {
        const float loss = t >= 0 ? lse - z : NAN;   // a target outside the vocabulary
        a.lse[j] = lse;
        if (a.reduction == FA2_REDUCE_NONE)
            a.loss[a.rowmap[j]] = loss;
        else
            a.row_loss[j] = loss;
    }
}

// none: zeros for the tokens that do not count.
__global__ __launch_bounds__(256) void xent_ignored_kernel(const XentArgs a) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < a.rows; i += (int64_t)gridDim.x * 256)
        if (a.pos[i] < 0) a.loss[i] = 0.f;
}

// sum, mean: one workgroup adds the rows' losses in a fixed order.
__global__ __launch_bounds__(1024) void xent_sum_kernel(const XentArgs a) {
    __shared__ double s[16];
    const int n = a.count[0];
    double v = 0.;
    for (int j = threadIdx.x; j < n; j += 1024) v += a.row_loss[j];
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o);
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < 16; ++i) v += s[i];
        a.loss[0] = (float)(a.reduction == FA2_REDUCE_MEAN ? v / n : v);   // mean of none: 0 / 0, as torch
    }
}

// ---------------------------------------------------------------------------
// Backward
// ---------------------------------------------------------------------------

// Factors of the rows of P, and the factor of the finished products.  sum and
// mean: every row has P_SCALE; none: the row's gradient over the largest one.
__global__ __launch_bounds__(1024) void xent_coef_kernel(const XentArgs a) {
    __shared__ float s[16];
    const int n = a.count[0];
    float top = 0.f;
    if (a.reduction == FA2_REDUCE_NONE) {
        for (int j = threadIdx.x; j < n; j += 1024) {
            const float v = fabsf(a.g[(int64_t)a.rowmap[j] * a.g_stride]);
            top = (v > top || v != v) ? v : top;
        }
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) {
            const float v = __shfl_xor(top, o);
            top = (v > top || v != v) ? v : top;
        }
        if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = top;
        __syncthreads();
        top = 0.f;
        for (int i = 0; i < 16; ++i) top = (s[i] > top || s[i] != s[i]) ? s[i] : top;
    }
    for (int j = threadIdx.x; j < a.rows_pad; j += 1024) {
        float f = 0.f;
        if (j < n) {
            f = P_SCALE;
            if (a.reduction == FA2_REDUCE_NONE) {
                const float v = a.g[(int64_t)a.rowmap[j] * a.g_stride];
                f = v == 0.f ? 0.f : v / top * P_SCALE;
            }
            if (a.tgt[j] < 0) f = NAN;
        }
        a.coef[j] = f;
    }
    if (threadIdx.x == 0) {
        const float u = a.reduction == FA2_REDUCE_NONE ? top : a.reduction == FA2_REDUCE_MEAN ? a.g[0] / (float)n : a.g[0];
        a.unscale[0] = n ? u / P_SCALE : 0.f;
    }
}

// A tile of P: logits again, softmax, minus one at the target, times the row's factor.
template <typename T>
__global__ __launch_bounds__(256) void xent_p_kernel(const XentArgs a) {
    __shared__ TileMem<T> s;
    const int nr = a.rows_pad / TN;
    const int rb = blockIdx.x % nr, vt = blockIdx.x / nr;
    const int n = a.count[0];
    const int lane = threadIdx.x & 63, c = lane & 31, g2 = lane >> 5;
    const int wm = (threadIdx.x >> 6 & 1) * 64, wn = (threadIdx.x >> 7) * 64;
    f16x acc[2][2];
    if (rb * TN < n) {
        const Operand<T> A = {static_cast<const T *>(a.w), a.w_stride, a.v0 + vt * TM, a.V, 0};
        const Operand<T> B = {static_cast<const T *>(a.xc), a.dp, rb * TN, a.rows_pad, 0};
        product_tile<T, true, true>(A, B, 0, a.dp, s, acc);
    } else if (rb * TN >= (n + XENT_PAD - 1) / XENT_PAD * XENT_PAD) {
        return;   // no product reads these rows
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int row = rb * TN + wn + 32 * j + c;
        const bool in = row < n;
        const float lse = in ? a.lse[row] : 0.f, f = in ? a.coef[row] : 0.f;
        const int t = in ? a.tgt[row] - a.v0 - vt * TM : -1;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                f4 v;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int r = 4 * q + e, mm = wm + 32 * i + acc_row(r, g2);
                    const float p = __expf(acc[i][j][r] - lse) - (mm == t ? 1.f : 0.f);
                    v[e] = in && a.v0 + vt * TM + mm < a.V && f != 0.f ? p * f : 0.f;
                }
                T *o = static_cast<T *>(a.P) + (int64_t)row * a.piece + vt * TM + wm + 32 * i + 8 * q + 4 * g2;
                *reinterpret_cast<typename vec_of<T>::v4 *>(o) = __builtin_convertvector(v, typename vec_of<T>::v4);
            }
    }
}

// dW of the piece: M side hidden columns, N side vocabulary rows, K packed tokens.
template <typename T>
__global__ __launch_bounds__(256) void xent_dw_kernel(const XentArgs a) {
    __shared__ TileMem<T> s;
    const int nd = (a.d + TM - 1) / TM;
    const int db = blockIdx.x % nd, vb = blockIdx.x / nd;
    const int n = a.count[0], kn = (n + XENT_PAD - 1) / XENT_PAD * XENT_PAD;
    const int lane = threadIdx.x & 63, c = lane & 31, g2 = lane >> 5;
    const int wm = (threadIdx.x >> 6 & 1) * 64, wn = (threadIdx.x >> 7) * 64;
    const Operand<T> A = {static_cast<const T *>(a.xc), a.dp, db * TM, a.dp, a.rows_pad};
    const Operand<T> B = {static_cast<const T *>(a.P), a.piece, vb * TN, a.piece, a.rows_pad};
    f16x acc[2][2];
    product_tile<T, false, false>(A, B, 0, kn, s, acc);
    const float u = a.unscale[0];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int v = a.v0 + vb * TN + wn + 32 * j + c;
        if (v >= a.v1) continue;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int col = db * TM + wm + 32 * i + acc_row(r, g2);
                if (col < a.d) static_cast<T *>(a.dw)[(int64_t)v * a.d + col] = (T)(acc[i][j][r] * u);
            }
    }
}

// The piece's share of dx: M side hidden columns, N side packed tokens, K a slice
// of the piece.
template <typename T>
__global__ __launch_bounds__(256) void xent_dx_kernel(const XentArgs a) {
    __shared__ TileMem<T> s;
    const int nd = (a.d + TM - 1) / TM, nr = a.rows_pad / TN;
    const int db = blockIdx.x % nd, rb = blockIdx.x / nd % nr, ks = blockIdx.x / nd / nr;
    if (rb * TN >= a.count[0]) return;
    const int lane = threadIdx.x & 63, c = lane & 31, g2 = lane >> 5;
    const int wm = (threadIdx.x >> 6 & 1) * 64, wn = (threadIdx.x >> 7) * 64;
    const int kt = (a.v1 - a.v0 + TK - 1) / TK;
    const int k0 = (int)((int64_t)kt * ks / a.ksplit) * TK, k1 = (int)((int64_t)kt * (ks + 1) / a.ksplit) * TK;
    const Operand<T> A = {static_cast<const T *>(a.w) + (int64_t)a.v0 * a.w_stride, a.w_stride, db * TM, a.dp, a.V - a.v0};
    const Operand<T> B = {static_cast<const T *>(a.P), a.piece, rb * TN, a.rows_pad, 0};
    f16x acc[2][2];
    product_tile<T, false, true>(A, B, k0, k1, s, acc);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        float *o = a.acc + ((int64_t)ks * a.rows_pad + rb * TN + wn + 32 * j + c) * a.d;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int col = db * TM + wm + 32 * i + acc_row(r, g2);
                if (col < a.d) o[col] = a.first ? acc[i][j][r] : o[col] + acc[i][j][r];
            }
    }
}

// dx of every token: the slices' sums, rounded once; zeros where a token does not count.
template <typename T>
__global__ __launch_bounds__(256) void xent_dx_out_kernel(const XentArgs a) {
    const int64_t total = a.rows * a.d;
    for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x; e < total; e += (int64_t)gridDim.x * 256) {
        const int64_t i = e / a.d;
        const int c = (int)(e - i * a.d), j = a.pos[i];
        float v = 0.f;
        if (j >= 0) {
            for (int s = 0; s < a.ksplit; ++s) v += a.acc[((int64_t)s * a.rows_pad + j) * a.d + c];
            v *= a.unscale[0];
        }
        static_cast<T *>(a.dx)[e] = (T)v;
    }
}

#define FA2_LAUNCH(kernel, grid, block)                                    \
    do {                                                                   \
        hipLaunchKernelGGL(kernel, dim3(grid), dim3(block), 0, st, a);     \
        const hipError_t e = hipGetLastError();                            \
        if (e != hipSuccess) return e;                                     \
    } while (0)

template <typename T>
hipError_t fwd(const XentArgs &a, hipStream_t st) {
    FA2_LAUNCH(xent_stats_kernel<T>, a.rows_pad / TN * a.splits, 256);
    if (a.reduction == FA2_REDUCE_NONE && a.rows > 0)
        FA2_LAUNCH(xent_ignored_kernel, (unsigned)((a.rows + 255) / 256 < 4096 ? (a.rows + 255) / 256 : 4096), 256);
    FA2_LAUNCH(xent_join_kernel<T>, a.rows_pad / 4, 256);
    if (a.reduction != FA2_REDUCE_NONE) FA2_LAUNCH(xent_sum_kernel, 1, 1024);
    return hipSuccess;
}

template <typename T>
hipError_t piece(const XentArgs &a, hipStream_t st) {
    const int nr = a.rows_pad / TN, nd = (a.d + TM - 1) / TM, nv = (a.v1 - a.v0 + TM - 1) / TM;
    FA2_LAUNCH(xent_p_kernel<T>, nr * nv, 256);
    if (a.dw) FA2_LAUNCH(xent_dw_kernel<T>, nd * nv, 256);
    if (a.dx) FA2_LAUNCH(xent_dx_kernel<T>, nd * nr * a.ksplit, 256);
    return hipSuccess;
}

}  // namespace

hipError_t launch_xent_pack(const XentArgs &a, hipStream_t st) {
    FA2_LAUNCH(xent_scan_kernel, 1, 1024);
    if (a.type == FA2_F16)
        FA2_LAUNCH(xent_pack_kernel<_Float16>, a.rows_pad / 4, 256);
    else
        FA2_LAUNCH(xent_pack_kernel<__bf16>, a.rows_pad / 4, 256);
    return hipSuccess;
}

hipError_t launch_xent_pad_weight(const void *w, int64_t w_stride, void *out, int V, int d, int dp, int type, hipStream_t st) {
    const dim3 grid(V < 4096 ? V : 4096), block(256);
    if (type == FA2_F16)
        hipLaunchKernelGGL(xent_pad_weight_kernel<_Float16>, grid, block, 0, st, static_cast<const _Float16 *>(w), w_stride,
                           static_cast<_Float16 *>(out), V, d, dp);
    else
        hipLaunchKernelGGL(xent_pad_weight_kernel<__bf16>, grid, block, 0, st, static_cast<const __bf16 *>(w), w_stride,
                           static_cast<__bf16 *>(out), V, d, dp);
    return hipGetLastError();
}

hipError_t launch_xent_fwd(const XentArgs &a, hipStream_t st) {
    return a.type == FA2_F16 ? fwd<_Float16>(a, st) : fwd<__bf16>(a, st);
}

hipError_t launch_xent_bwd_prepare(const XentArgs &a, hipStream_t st) {
    FA2_LAUNCH(xent_coef_kernel, 1, 1024);
    return hipSuccess;
}

hipError_t launch_xent_bwd_piece(const XentArgs &a, hipStream_t st) {
    return a.type == FA2_F16 ? piece<_Float16>(a, st) : piece<__bf16>(a, st);
}

hipError_t launch_xent_bwd_finish(const XentArgs &a, hipStream_t st) {
    const int64_t want = (a.rows * a.d + 255) / 256;
    const unsigned grid = (unsigned)(want < 8192 ? want : 8192);
    if (a.type == FA2_F16)
        FA2_LAUNCH(xent_dx_out_kernel<_Float16>, grid, 256);
    else
        FA2_LAUNCH(xent_dx_out_kernel<__bf16>, grid, 256);
    return hipSuccess;
}

}  // namespace fa2
