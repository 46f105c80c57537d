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
// which is complete, and the piece's share of dx, summed in fp32.  P of the next
// piece goes beside dW and dx of this one, into a second scratch.
//
// Tokens that do not count are taken out first (packed rows), so that no product
// works on them and nothing in their states, inf and NaN included, reaches a result.
//
// Rounding P to 16 bits (its relative error is at most half a step, and the
// errors of a sum's many terms are independent) keeps both gradient products on
// the matrix units; the gradients themselves are rounded to the same type.  P is
// scaled so that its largest possible value is 2^15: in fp16 probabilities down
// to 2^-29 stay normal numbers.
#include <type_traits>

#include "fa2_product.h"

namespace fa2 {
namespace {

constexpr float P_SCALE = 32768.f;

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
// Each lane keeps a reference r and the sum of exp(z - r) of the logits it has
// seen.  r is the maximum of the lane's first tile and moves only when a sum
// passes 2^100: fp32 holds the terms of any larger logits until then.  The slice's
// tiles are one stream of stages: the next tile's transfers run behind the
// exponentials.
template <typename T, int NP, int WM, int WN>
__global__ __launch_bounds__(512, 2) void xent_stats_kernel(const XentArgs a) {
    typedef Product<T, true, true, 4, NP, WM, WN> Pr;
    constexpr int MI = Pr::MI, NI = Pr::NI;
    __shared__ __align__(16) char mem[Pr::LDS];
    const int nr = a.rows_pad / Pr::TN;
    const int rb = blockIdx.x % nr, split = blockIdx.x / nr;
    if (rb * Pr::TN >= a.count[0]) return;
    const int tiles = (a.V + Pr::TM - 1) / Pr::TM;
    const int t0 = (int)((int64_t)tiles * split / a.splits), t1 = (int)((int64_t)tiles * (split + 1) / a.splits);
    const int lane = threadIdx.x & 63, c = lane & 31, g2 = lane >> 5;
    Pr pr;
    pr.init(mem);
    pr.A.init(a.w, a.w_stride, t0 * Pr::TM, a.V, 0);
    pr.B.init(a.xc, a.dp, rb * Pr::TN, a.rows_pad, 0);
    float ref[NI], sum[NI];
#pragma unroll
    for (int j = 0; j < NI; ++j) {
        ref[j] = -INFINITY;
        sum[j] = 0.f;
    }
    int nt = t0, nk = 0;   // tile and k of the next stage
    auto next = [&](int buf) FA2_INLINE {
        if (nt >= t1) return;
        pr.issue(nk, buf);
        nk += PK;
        if (nk == a.dp) {
            nk = 0;
            if (++nt < t1) pr.A.init(a.w, a.w_stride, nt * Pr::TM, a.V, 0);
        }
    };
    pr.begin(next);
    for (int t = t0; t < t1; ++t) {
        f16x acc[MI][NI];
        pr.zero(acc);
        pr.steps(a.dp / PK, acc, next);
        // Rows of this wave's part that are past the vocabulary (in the last tile) are left out.
        const int left = a.V - t * Pr::TM - pr.wm;
        auto add_tile = [&](auto tail, int j) FA2_INLINE {
            constexpr bool TAIL = decltype(tail)::value;
            auto in = [&](int i, int r) FA2_INLINE { return !TAIL || 32 * i + acc_row(r, g2) < left; };
            auto tile_sum = [&](float r0, float s, float log2e) FA2_INLINE {
                const float sub = r0 * log2e;
#pragma unroll
                for (int i = 0; i < MI; ++i) {
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const float e = __builtin_amdgcn_exp2f(acc[i][j][r] * log2e - sub);
                        s += in(i, r) ? e : 0.f;
                    }
                    asm volatile("" : "+v"(s));   // one block's exponentials at a time: all at once spill
                }
                return s;
            };
            float s = tile_sum(ref[j] == -INFINITY ? 0.f : ref[j], sum[j], LOG2E);
            if (__any(ref[j] == -INFINITY || !(s < 0x1p100f))) {
                FA2_COLD_BRANCH();
                float top = ref[j];
#pragma unroll
                for (int i = 0; i < MI; ++i)
#pragma unroll
                    for (int r = 0; r < 16; ++r) top = in(i, r) ? fmaxf(top, acc[i][j][r]) : top;
                const float base = top == -INFINITY ? 0.f : top;
                float log2e = LOG2E;
                asm volatile("" : "+v"(log2e));   // keeps the first sum's products from being held for this one
                s = tile_sum(base, sum[j] * __builtin_amdgcn_exp2f((ref[j] - base) * LOG2E), log2e);
                ref[j] = top;
            }
            sum[j] = s;
        };
        if (left >= Pr::TM / WM) {
#pragma unroll
            for (int j = 0; j < NI; ++j) add_tile(std::false_type(), j);
        } else {
            FA2_COLD_BRANCH();
#pragma unroll
            for (int j = 0; j < NI; ++j) add_tile(std::true_type(), j);
        }
    }
    lds_barrier();
    // Lanes, then the waves along the vocabulary (the panels are no longer read).
    float *jm = reinterpret_cast<float *>(mem), *jl = jm + WM * Pr::TN;
#pragma unroll
    for (int j = 0; j < NI; ++j) {
        join_max_sum(ref[j], sum[j], __shfl_xor(ref[j], 32), __shfl_xor(sum[j], 32));
        if (g2 == 0) {
            const int at = pr.wm / (Pr::TM / WM) * Pr::TN + pr.wn + 32 * j + c;
            jm[at] = ref[j];
            jl[at] = sum[j];
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < Pr::TN; i += 512) {
        float m = jm[i], l = jl[i];
#pragma unroll
        for (int w = 1; w < WM; ++w) join_max_sum(m, l, jm[w * Pr::TN + i], jl[w * Pr::TN + i]);
        *(reinterpret_cast<f2 *>(a.part) + (int64_t)split * a.rows_pad + rb * Pr::TN + i) = f2{m, l};
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

// The work of one launch of the backward: dW and dx of a piece, and P of the piece
// after it, as items of one grid, the long ones first; P's many short items fill the
// compute units that the others leave.  Lengths are in stages of 64 k.
struct XentWork {
    int rt;            // tiles of 256 tokens that count
    int dw, dx, p;     // items
    int xs;            // slices of dx's k
};

constexpr int P_STRIP = 4;       // tiles of P an item
constexpr int P_TILE_EXTRA = 4;  // stages that the softmax of a tile of P takes as long as

__device__ __forceinline__ XentWork xent_work(const XentArgs &a, int n) {
    XentWork k;
    const int nd = (a.d + 255) / 256, nv = (a.v1 - a.v0 + 255) / 256, nvp = (a.p1 - a.p0 + 255) / 256;
    k.rt = (n + 255) / 256;
    // Slices of dx: no longer than three quarters of a compute unit's share of a
    // launch (with pieces of full width; the same number for every piece).
    const int64_t full = a.piece / 256;
    const int64_t total = full * k.rt * (nd * 8 + (a.pieces > 1 ? a.dp / PK + P_TILE_EXTRA : 0));
    const int share = (int)max((int64_t)4, total * 3 / (4 * 256));
    k.xs = max(1, min((a.piece / PK + share - 1) / share, a.xcap / max(k.rt, 1)));
    k.dw = a.dw ? nd * nv * a.wsplit : 0;
    k.dx = a.dx && nv > 0 ? nd * k.rt * k.xs : 0;
    k.p = k.rt * ((nvp + P_STRIP - 1) / P_STRIP);
    return k;
}

// Workgroups go to the eight XCDs in turn: the l-th of n items, numbered so that an
// XCD's items are neighbours (their operands meet in its L2).
__device__ __forceinline__ int xcd_item(int l, int n) {
    const int x = l & 7;
    return x * (n >> 3) + min(x, n & 7) + (l >> 3);
}

// P_STRIP tiles of P: logits again, softmax, minus one at the target, times the row's
// factor; M side vocabulary rows, N side tokens.
template <typename T>
__device__ __forceinline__ void xent_p_item(const XentArgs &a, const XentWork &k, int item, int n, char *mem, char *out) {
    typedef Product<T, true, true, 4, 4, 2, 4> Pr;
    const int tiles = (a.p1 - a.p0 + 255) / 256, strips = (tiles + P_STRIP - 1) / P_STRIP;
    // groups of 8 token tiles, in a group the tokens fastest
    const int g = item / (8 * strips), gs = min(8, k.rt - 8 * g), in = item - g * 8 * strips;
    const int rb = 8 * g + in % gs, t0 = in / gs * P_STRIP, t1 = min(tiles, t0 + P_STRIP);
    const int lane = threadIdx.x & 63, c = lane & 31, g2 = lane >> 5;
    Pr pr;
    pr.init(mem);
    pr.A.init(a.w, a.w_stride, a.p0 + t0 * Pr::TM, a.V, 0);
    pr.B.init(a.xc, a.dp, rb * Pr::TN, a.rows_pad, 0);
    float f[Pr::NI], sub[Pr::NI];
    int tgt[Pr::NI];
#pragma unroll
    for (int j = 0; j < Pr::NI; ++j) {
        const int row = rb * Pr::TN + pr.wn + 32 * j + c;
        f[j] = a.coef[row];
        sub[j] = row < n ? a.lse[row] * LOG2E : 0.f;
        tgt[j] = a.tgt[row] - pr.wm;
    }
    int nt = t0, nk = 0;
    auto next = [&](int buf) FA2_INLINE {
        if (nt >= t1) return;
        pr.issue(nk, buf);
        nk += PK;
        if (nk == a.dp) {
            nk = 0;
            if (++nt < t1) pr.A.init(a.w, a.w_stride, a.p0 + nt * Pr::TM, a.V, 0);
        }
    };
    pr.begin(next);
    char *blk = out + (threadIdx.x >> 6) * 4096;
    for (int t = t0; t < t1; ++t) {
        const int v0 = a.p0 + t * Pr::TM;
        f16x acc[Pr::MI][Pr::NI];
        pr.zero(acc);
        pr.steps(a.dp / PK, acc, next);
#pragma unroll
        for (int j = 0; j < Pr::NI; ++j) {
            T *o = static_cast<T *>(a.Pn) + (int64_t)(rb * Pr::TN + pr.wn + 32 * j) * a.piece + t * Pr::TM + pr.wm;
#pragma unroll
            for (int i = 0; i < Pr::MI; i += 2) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const float p = __builtin_amdgcn_exp2f(acc[i + h][j][r] * LOG2E - sub[j]) * f[j];
                        acc[i + h][j][r] = f[j] != 0.f ? p : 0.f;
                    }
                    const int at = tgt[j] - v0 - 32 * (i + h);
                    if (__any(at >= 0 && at < 32)) {
                        FA2_COLD_BRANCH();
#pragma unroll
                        for (int r = 0; r < 16; ++r)
                            if (at == acc_row(r, g2)) acc[i + h][j][r] -= f[j];
                    }
                    if (v0 + pr.wm + 32 * (i + h) + 32 > a.V) {   // rows past the vocabulary
                        FA2_COLD_BRANCH();
#pragma unroll
                        for (int r = 0; r < 16; ++r)
                            if (v0 + pr.wm + 32 * (i + h) + acc_row(r, g2) >= a.V) acc[i + h][j][r] = 0.f;
                    }
                }
                store_rows<T>(acc[i][j], acc[i + 1][j], 1.f, blk, o + 32 * i, a.piece, 32, 64, true);
            }
        }
    }
}

// A tile of the piece's dW, or of a slice of its k: M side hidden columns, N side
// vocabulary rows, K packed tokens.
template <typename T>
__device__ __forceinline__ void xent_dw_item(const XentArgs &a, int item, int n, char *mem) {
    typedef Product<T, false, false, 4, 4, 2, 4> Pr;
    const int nd = (a.d + 255) / 256, nv = (a.v1 - a.v0 + 255) / 256;
    const int db = item % nd, vb = item / nd % nv, s = item / nd / nv;
    const int kt = (n + 255) / 256 * (256 / PK);
    const int k0 = (int)((int64_t)kt * s / a.wsplit) * PK, k1 = (int)((int64_t)kt * (s + 1) / a.wsplit) * PK;
    Pr pr;
    pr.init(mem);
    pr.A.init(a.xc, a.dp, db * Pr::TM, a.dp, a.rows_pad);
    pr.B.init(a.P, a.piece, vb * Pr::TN, a.piece, a.rows_pad);
    f16x acc[Pr::MI][Pr::NI];
    pr.run(k0, k1, acc);
    const int lane = threadIdx.x & 63, c = lane & 31, g2 = lane >> 5;
    const float u = a.unscale[0];
    char *blk = mem + (threadIdx.x >> 6) * 4096;
#pragma unroll
    for (int j = 0; j < Pr::NI; ++j) {
        const int v = vb * Pr::TN + pr.wn + 32 * j;   // of the piece
#pragma unroll
        for (int i = 0; i < Pr::MI; i += 2) {
            const int col = db * Pr::TM + pr.wm + 32 * i;
            if (a.wsplit == 1) {
                store_rows<T>(acc[i][j], acc[i + 1][j], u, blk, static_cast<T *>(a.dw) + (int64_t)(a.v0 + v) * a.d + col, a.d,
                              a.v1 - a.v0 - v, a.d - col, a.d % 8 == 0);
            } else {   // rows of the slice's sums: [wsplit][piece][dp], four columns a store
                float *o = a.wacc + ((int64_t)s * a.piece + v + c) * a.dp + col;
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        if (col + 32 * h < a.dp) {
                            f4 x;
#pragma unroll
                            for (int e = 0; e < 4; ++e) x[e] = acc[i + h][j][4 * q + e];
                            *reinterpret_cast<f4 *>(o + 32 * h + 8 * q + 4 * g2) = x;
                        }
            }
        }
    }
}

// A tile of the piece's share of dx, or of a slice of its k: M side packed tokens, N
// side hidden columns, K the piece.
template <typename T>
__device__ __forceinline__ void xent_dx_item(const XentArgs &a, const XentWork &k, int item, char *mem) {
    typedef Product<T, true, false, 4, 4, 2, 4> Pr;
    const int nd = (a.d + 255) / 256;
    const int db = item % nd, rb = item / nd % k.rt, s = item / nd / k.rt;
    const int kt = (a.v1 - a.v0 + PK - 1) / PK;
    const int k0 = (int)((int64_t)kt * s / k.xs) * PK, k1 = (int)((int64_t)kt * (s + 1) / k.xs) * PK;
    Pr pr;
    pr.init(mem);
    pr.A.init(a.P, a.piece, rb * Pr::TM, a.rows_pad, 0);
    pr.B.init(static_cast<const T *>(a.w) + (int64_t)a.v0 * a.w_stride, a.w_stride, db * Pr::TN, a.dp, a.V - a.v0);
    f16x acc[Pr::MI][Pr::NI];
    pr.run(k0, k1, acc);
    const int lane = threadIdx.x & 63, c = lane & 31, g2 = lane >> 5;
#pragma unroll
    for (int j = 0; j < Pr::NI; ++j) {
        const int col = db * Pr::TN + pr.wn + 32 * j + c;
        if (col >= a.d) continue;
#pragma unroll
        for (int i = 0; i < Pr::MI; ++i) {
            float *o = a.acc + ((int64_t)(s * k.rt + rb) * Pr::TM + pr.wm + 32 * i) * a.d + col;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                float *q = o + (int64_t)acc_row(r, g2) * a.d;
                *q = a.v0 == 0 ? acc[i][j][r] : *q + acc[i][j][r];
            }
        }
    }
}

template <typename T>
__global__ __launch_bounds__(512, 2) void xent_grad_kernel(const XentArgs a) {
    constexpr int PANELS = Product<T, true, true, 4, 4, 2, 4>::LDS;
    __shared__ __align__(16) char mem[PANELS + 8 * 4096];
    const int n = a.count[0];
    const XentWork k = xent_work(a, n);
    int l = blockIdx.x;
    const bool dw_first = (int64_t)k.rt * 4 * k.xs * PK > (int64_t)(a.v1 - a.v0) * a.wsplit;   // the longer ones
    if (dw_first && l < k.dw) return xent_dw_item<T>(a, xcd_item(l, k.dw), n, mem);
    l -= dw_first ? k.dw : 0;
    if (l < k.dx) return xent_dx_item<T>(a, k, xcd_item(l, k.dx), mem);
    l -= k.dx;
    if (!dw_first && l < k.dw) return xent_dw_item<T>(a, xcd_item(l, k.dw), n, mem);
    l -= dw_first ? 0 : k.dw;
    if (l < k.p) xent_p_item<T>(a, k, xcd_item(l, k.p), n, mem, mem + PANELS);
}

// dW of a piece whose k was sliced: the slices' sums in order.
template <typename T>
__global__ __launch_bounds__(256) void xent_dw_join_kernel(const XentArgs a) {
    const float u = a.unscale[0];
    const int64_t total = (int64_t)(a.v1 - a.v0) * a.d;
    for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x; e < total; e += (int64_t)gridDim.x * 256) {
        const int64_t v = e / a.d;
        const int c = (int)(e - v * a.d);
        float x = 0.f;
        for (int s = 0; s < a.wsplit; ++s) x += a.wacc[((int64_t)s * a.piece + v) * a.dp + c];
        static_cast<T *>(a.dw)[(int64_t)a.v0 * a.d + e] = (T)(x * u);
    }
}

// dx of every token: the slices' sums, rounded once; zeros where a token does not count.
template <typename T>
__global__ __launch_bounds__(256) void xent_dx_out_kernel(const XentArgs a) {
    const int64_t total = a.rows * a.d;
    const XentWork k = xent_work(a, a.count[0]);
    for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x; e < total; e += (int64_t)gridDim.x * 256) {
        const int64_t i = e / a.d;
        const int c = (int)(e - i * a.d), j = a.pos[i];
        float v = 0.f;
        if (j >= 0) {
            for (int s = 0; s < k.xs; ++s) v += a.acc[((int64_t)s * k.rt * 256 + j) * a.d + c];
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
    if (a.narrow)
        FA2_LAUNCH((xent_stats_kernel<T, 1, 8, 1>), a.rows_pad / 64 * a.splits, 512);
    else
        FA2_LAUNCH((xent_stats_kernel<T, 4, 2, 4>), a.rows_pad / 256 * a.splits, 512);
    if (a.reduction == FA2_REDUCE_NONE && a.rows > 0)
        FA2_LAUNCH(xent_ignored_kernel, (unsigned)((a.rows + 255) / 256 < 4096 ? (a.rows + 255) / 256 : 4096), 256);
    FA2_LAUNCH(xent_join_kernel<T>, a.rows_pad / 4, 256);
    if (a.reduction != FA2_REDUCE_NONE) FA2_LAUNCH(xent_sum_kernel, 1, 1024);
    return hipSuccess;
}

// P of [p0, p1) beside dW and dx of [v0, v1); either may be empty.
template <typename T>
hipError_t grad(const XentArgs &a, hipStream_t st) {
    const int rt = a.rows_pad / 256, nd = (a.d + 255) / 256, nv = (a.v1 - a.v0 + 255) / 256, np = (a.p1 - a.p0 + 255) / 256;
    const int items = nd * nv * a.wsplit + (nv ? nd * a.xcap : 0) + rt * ((np + P_STRIP - 1) / P_STRIP);   // the most there can be
    FA2_LAUNCH(xent_grad_kernel<T>, items, 512);
    if (nv && a.dw && a.wsplit > 1) {
        const int64_t want = ((int64_t)(a.v1 - a.v0) * a.d + 255) / 256;
        FA2_LAUNCH(xent_dw_join_kernel<T>, (unsigned)(want < 8192 ? want : 8192), 256);
    }
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

hipError_t launch_xent_grad(const XentArgs &a, hipStream_t st) {
    return a.type == FA2_F16 ? grad<_Float16>(a, st) : grad<__bf16>(a, st);
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
