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
#include "fa2_product.h"

namespace fa2 {
namespace {

constexpr float P_SCALE = 32768.f;

// Elements of XentArgs::count.
enum { N_TOKENS = 0, STAT_SPLITS = 1 };

// ---------------------------------------------------------------------------
// Packing
// ---------------------------------------------------------------------------

constexpr int PACK_ROWS = 64;   // packed rows a workgroup has at a time, at most

// Every workgroup counts through all targets, and does its share of the rest: the
// packed rows' token, target and states (zeros behind the last column and up to a
// whole tile of rows), and the tokens' packed rows.  Counting everywhere takes no
// second launch and no memory between workgroups: 16384 tokens x 768 in 20 us, of which
// the copy of the states is half (50 MB); read once a workgroup, the targets come
// from L2.
template <typename T>
__global__ __launch_bounds__(1024) void xent_pack_kernel(const XentArgs a) {
    constexpr int Q = 16;                // targets a thread has at a time
    __shared__ int before[16 * Q + 1];   // tokens that count in each run of 64 targets; then, before it
    __shared__ int src[PACK_ROWS];
    typedef typename vec_of<T>::v8 v8;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int share = ((int)a.rows + gridDim.x - 1) / gridDim.x;   // of the tokens' packed rows (at most 2^24 tokens)
    const int rows_n = (int)a.rows, i0 = blockIdx.x * share, i1 = min(rows_n, i0 + share);
    const bool vec = a.x_stride % 8 == 0 && (reinterpret_cast<uintptr_t>(a.x) & 15) == 0 && a.d % 8 == 0;
    for (int j0 = blockIdx.x * a.pack_rows; j0 < a.rows_pad; j0 += gridDim.x * a.pack_rows) {
        int n = 0;   // tokens that count so far
        for (int r0 = 0; r0 < rows_n; r0 += 1024 * Q) {
            const int qs = min(Q, (rows_n - r0 + 1023) / 1024);   // in use
            const int first = r0 + (int)threadIdx.x;              // run 16 q + wave: targets r0 + 1024 q + 64 wave ..
            int64_t t[Q];
            uint64_t m[Q];
#pragma unroll
            for (int q = 0; q < Q; ++q)
                if (q < qs) t[q] = first + q * 1024 < rows_n ? a.target[first + q * 1024] : a.ignore;
#pragma unroll
            for (int q = 0; q < Q; ++q)
                if (q < qs) {
                    m[q] = __ballot(first + q * 1024 < rows_n && t[q] != a.ignore);
                    if (lane == 0) before[16 * q + wave] = __popcll(m[q]);
                }
            __syncthreads();
            if (wave == 0) {   // exclusive sums over the runs, four a lane
                int c[4], sum = 0;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    c[k] = 4 * lane + k < 16 * qs ? before[4 * lane + k] : 0;
                    sum += c[k];
                }
                int up = sum;
#pragma unroll
                for (int o = 1; o < 64; o <<= 1) {
                    const int v = __shfl_up(up, o);
                    up += lane >= o ? v : 0;
                }
                int at = n + up - sum;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    before[4 * lane + k] = at;
                    at += c[k];
                }
                if (lane == 63) before[16 * Q] = at;
            }
            __syncthreads();
#pragma unroll
            for (int q = 0; q < Q; ++q)
                if (q < qs) {
                    const int i = first + q * 1024;
                    const bool in = m[q] >> lane & 1;
                    const int j = before[16 * q + wave] + __popcll(m[q] & ((1ull << lane) - 1));
                    if (i >= i0 && i < i1) a.pos[i] = in ? j : -1;
                    if (in && j >= j0 && j < j0 + a.pack_rows) {
                        src[j - j0] = i;
                        a.rowmap[j] = i;
                        a.tgt[j] = t[q] >= 0 && t[q] < a.V ? (int)t[q] : -1;
                    }
                }
            n = before[16 * Q];
            __syncthreads();   // before is free
        }
        if (j0 == 0 && threadIdx.x == 0) {
            a.count[N_TOKENS] = n;
            a.count[STAT_SPLITS] = xent_stat_splits(a.stat_tile_n, a.stat_tile_m, a.stat_slots, a.stat_rounds, n, a.V);
        }
        if ((int)threadIdx.x < a.pack_rows && j0 + (int)threadIdx.x >= n) a.tgt[j0 + threadIdx.x] = -1;
        __syncthreads();
        // Wave w: rows w, w + 16, .., up to four at a time; 8 elements a lane.
        const int rows = min(a.pack_rows, (n + XENT_PAD - 1) / XENT_PAD * XENT_PAD - j0);
        for (int c = lane * 8; c < a.dp; c += 512) {
            v8 v[PACK_ROWS / 16];
#pragma unroll
            for (int q = 0; q < PACK_ROWS / 16; ++q) {
                const int r = wave + 16 * q;
                v[q] = v8{};
                if (r < rows && j0 + r < n) {
                    const T *x = static_cast<const T *>(a.x) + (int64_t)src[r] * a.x_stride;
                    if (vec) {
                        if (c < a.d) v[q] = *reinterpret_cast<const v8 *>(x + c);
                    } else {
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            if (c + e < a.d) v[q][e] = x[c + e];
                    }
                }
            }
#pragma unroll
            for (int q = 0; q < PACK_ROWS / 16; ++q) {
                const int r = wave + 16 * q;
                if (r < rows) *reinterpret_cast<v8 *>(static_cast<T *>(a.xc) + (int64_t)(j0 + r) * a.dp + c) = v[q];
            }
        }
        __syncthreads();   // src is free
    }
}

// Copy of the weight with rows of dp elements, for hidden sizes that 16-byte loads do
// not divide.
template <typename T>
__global__ __launch_bounds__(256) void xent_pad_weight_kernel(const T *w, int64_t stride, T *out, int V, int d, int dp) {
    for (int64_t r = blockIdx.x; r < V; r += gridDim.x)
        for (int c = threadIdx.x; c < dp; c += 256) out[r * dp + c] = c < d ? w[r * stride + c] : (T)0.f;
}

// Workgroups go to the eight XCDs in turn: the l-th of n items, numbered so that an
// XCD's items are neighbours (their operands meet in its L2).
__device__ __forceinline__ int xcd_item(int l, int n) {
    const int x = l & 7;
    return x * (n >> 3) + min(x, n & 7) + (l >> 3);
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

// Maximum and sum of exp of each packed row over a slice of the vocabulary.  The M
// side are vocabulary rows, the N side tokens: a lane holds one token's logits.  Each
// lane keeps a reference r and the sum of exp(z - r) of the logits it has seen.  r is
// the maximum of the lane's first tile and moves only when a sum passes 2^100: fp32
// holds the terms of any larger logits until then.  The slice's tiles are one stream
// of stages: the next tile's transfers run behind the exponentials.
//
// Bound by the matrix units at the board's power: 16384 tokens x 32000 x 768 in fp16
// take 710 us, 1134 TFLOP/s, where a library product of 8192^3 reaches 1215 and both keep
// the units busy in the same number of cycles a second.  Eight waves of 128 x 64 (four
// of 128 x 128 with their accumulators in AGPRs: 6% slower over 8 x 1023 tokens).  Few
// tokens: 199 x 32000 x 768 take 16.4 us, of which the weights' 49 MB are 10; the rest is
// one tile's start and end, which 250 workgroups cannot hide behind another's.
template <typename T, Source W, int MP, int NP, int WM, int WN, int NS>
__global__ __launch_bounds__(512, 2) void xent_stats_kernel(const XentArgs a) {
    typedef Product<T, true, true, W, MP == 4 ? PADDED : W, MP, NP, WM, WN, NS> Pr;   // MP < 4: the states may be the caller's
    constexpr int MI = Pr::MI, NI = Pr::NI;
    __shared__ __align__(16) char mem[Pr::LDS];
    const int n = a.direct ? (int)a.rows : a.count[N_TOKENS], splits = a.direct ? a.stat_splits : a.count[STAT_SPLITS];
    const int rt = (n + Pr::TN - 1) / Pr::TN;
    if ((int)blockIdx.x >= rt * splits) return;
    // groups of 8 token tiles, in a group the tokens fastest: a slice's weights meet in one
    // XCD's L2 (groups of 4: equal; of 16, here and for P: the whole training call 0.6 to 1% slower)
    const int item = xcd_item(blockIdx.x, rt * splits), g = item / (8 * splits), gs = min(8, rt - 8 * g), in_g = item - g * 8 * splits;
    const int rb = 8 * g + in_g % gs, split = in_g / gs;
    const int tiles = (a.V + Pr::TM - 1) / Pr::TM;
    const int t0 = (int)((int64_t)tiles * split / splits), t1 = (int)((int64_t)tiles * (split + 1) / splits);
    const int lane = threadIdx.x & 63, c = lane & 31, g2 = lane >> 5;
    Pr pr;
    pr.init(mem);
    pr.A.init(a.w, a.w_stride, t0 * Pr::TM, a.V, a.wd);
    pr.B.init(a.xc, a.xc_stride, rb * Pr::TN, a.direct ? n : a.rows_pad, a.direct ? a.wd : a.dp);
    float ref[NI], sum[NI];
#pragma unroll
    for (int j = 0; j < NI; ++j) {
        ref[j] = -INFINITY;
        sum[j] = 0.f;
    }
    int nt = t0, nk = 0;   // tile and k of the next stage
    auto next = [&](int buf) FA2_INLINE {
        if (nt >= t1) return false;
        pr.issue(nk, buf);
        nk += PK;
        if (nk == a.dp) {
            nk = 0;
            if (++nt < t1) pr.A.init(a.w, a.w_stride, nt * Pr::TM, a.V, a.wd);
        }
        return true;
    };
    typename Pr::Stream stream;
    pr.begin(stream, next);
    for (int t = t0; t < t1; ++t) {
        f16x acc[MI][NI];
        pr.steps(stream, a.dp / PK, acc, next);
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
            float s = INFINITY;   // the first tile has no reference yet
            if (t > t0) s = tile_sum(ref[j] == -INFINITY ? 0.f : ref[j], sum[j], LOG2E);
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
        reinterpret_cast<f2 *>(a.part)[(int64_t)(rb * Pr::TN + i) * splits + split] = f2{m, l};
    }
}

// One wave a token: joins its slices, and forms the target's logit as a product of its
// own (found among the tiles' logits it cost the forward's kernel 6%).
template <typename T>
__global__ __launch_bounds__(256) void xent_join_kernel(const XentArgs a) {
    const int lane = threadIdx.x & 63, splits = a.direct ? a.stat_splits : a.count[STAT_SPLITS];
    const int64_t i = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (i >= a.rows) return;
    const int64_t target = a.target[i];
    const int j = target == a.ignore ? -1 : a.direct ? (int)i : a.pos[i];
    float loss = 0.f;
    if (j >= 0) {
        const int t = target >= 0 && target < a.V ? (int)target : -1;
        // The first slices' pairs are on their way while the target's row is found and read.
        constexpr int FIRST = 4;
        const f2 *part = reinterpret_cast<const f2 *>(a.part) + (int64_t)j * splits;
        f2 p[FIRST];
#pragma unroll
        for (int q = 0; q < FIRST; ++q) p[q] = lane + 64 * q < splits ? part[lane + 64 * q] : f2{-INFINITY, 0.f};
        typedef typename vec_of<T>::v8 v8;
        const T *x = static_cast<const T *>(a.xc) + (int64_t)j * a.xc_stride;
        const T *w = static_cast<const T *>(a.w) + (int64_t)max(t, 0) * a.w_stride;
        float z = 0.f;
        for (int c = lane * 8; c < a.wd; c += 512) {
            const f8 xv = __builtin_convertvector(*reinterpret_cast<const v8 *>(x + c), f8);
            const f8 wv = __builtin_convertvector(*reinterpret_cast<const v8 *>(w + c), f8);
#pragma unroll
            for (int e = 0; e < 8; ++e) z += xv[e] * wv[e];
        }
        float m = -INFINITY, l = 0.f;
#pragma unroll
        for (int q = 0; q < FIRST; ++q) join_max_sum(m, l, p[q][0], p[q][1]);
        for (int s = lane + 64 * FIRST; s < splits; s += 64) join_max_sum(m, l, part[s][0], part[s][1]);
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) {
            join_max_sum(m, l, __shfl_xor(m, o), __shfl_xor(l, o));
            z += __shfl_xor(z, o);
        }
        const float lse = m + logf(l);
        loss = t >= 0 ? lse - z : NAN;   // a target outside the vocabulary
        if (lane == 0 && !a.direct) a.lse[j] = lse;
    }
    if (lane == 0) (a.reduction == FA2_REDUCE_NONE ? a.loss : a.row_loss)[i] = loss;
}

// sum, mean: one workgroup adds the tokens' losses in a fixed order.
__global__ __launch_bounds__(1024) void xent_sum_kernel(const XentArgs a) {
    __shared__ double sums[16];
    double v = 0.;
    for (int64_t i = threadIdx.x; i < a.rows; i += 1024) v += a.row_loss[i];
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o);
    if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = v;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int k = 1; k < 16; ++k) v += sums[k];
        a.loss[0] = (float)(a.reduction == FA2_REDUCE_MEAN ? v / a.count[N_TOKENS] : v);   // mean of none: 0 / 0, as torch
    }
}

// ---------------------------------------------------------------------------
// Backward
// ---------------------------------------------------------------------------

// none: each row of P is scaled by its gradient over the largest finite one, which the
// finished products are multiplied with.  (sum and mean: every row has 1.)  A gradient
// that is not finite makes its own row of dx not finite, and dW.
__global__ __launch_bounds__(1024) void xent_coef_kernel(const XentArgs a) {
    __shared__ float s[16];
    const int n = a.count[N_TOKENS];
    float top = 0.f;
    for (int j = threadIdx.x; j < n; j += 1024) {
        const float v = fabsf(a.g[(int64_t)a.rowmap[j] * a.g_stride]);
        top = v < INFINITY ? fmaxf(top, v) : top;
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = top;
    __syncthreads();
    top = 0.f;
    for (int i = 0; i < 16; ++i) top = fmaxf(top, s[i]);
    for (int j = threadIdx.x; j < n; j += 1024) {
        const float v = a.g[(int64_t)a.rowmap[j] * a.g_stride];
        a.coef[j] = v == 0.f ? 0.f : v / top;
    }
    if (threadIdx.x == 0) a.unscale[0] = top / P_SCALE;
}

// What the products of P are multiplied with.
__device__ __forceinline__ float xent_unscale(const XentArgs &a, int n) {
    if (n == 0) return 0.f;
    if (a.reduction == FA2_REDUCE_NONE) return a.unscale[0];
    return (a.reduction == FA2_REDUCE_MEAN ? a.g[0] / (float)n : a.g[0]) / P_SCALE;
}

// k.strip tiles of P: logits again, softmax, minus one at the target; M side
// vocabulary rows, N side tokens.  In units of 1 / P_SCALE, times the row's factor.
// Formed again, since keeping 16-bit logits would take their whole matrix: one
// product in four.  16384 tokens x 8192 columns x 768 alone: 210 us, 980 TFLOP/s.
template <typename T, Source W, int MP>
__device__ __forceinline__ void xent_p_item(const XentArgs &a, const XentWork &k, int item, int n, char *mem, char *out) {
    typedef Product<T, true, true, W, PADDED, MP, MP, 2, 4> Pr;
    const int tiles = (a.p1 - a.p0 + Pr::TM - 1) / Pr::TM, strips = (tiles + k.strip - 1) / k.strip;
    // groups of 8 token tiles, in a group the tokens fastest
    const int g = item / (8 * strips), gs = min(8, k.rt - 8 * g), in = item - g * 8 * strips;
    const int rb = 8 * g + in % gs, t0 = in / gs * k.strip, t1 = min(tiles, t0 + k.strip);
    const int lane = threadIdx.x & 63, c = lane & 31, g2 = lane >> 5;
    Pr pr;
    pr.init(mem);
    pr.A.init(a.w, a.w_stride, a.p0 + t0 * Pr::TM, a.V, a.wd);
    pr.B.init(a.xc, a.dp, rb * Pr::TN, a.rows_pad, a.dp);
    float f[Pr::NI], sub[Pr::NI];
    int tgt[Pr::NI];
#pragma unroll
    for (int j = 0; j < Pr::NI; ++j) {
        const int row = rb * Pr::TN + pr.wn + 32 * j + c;
        const int t = a.tgt[row];
        f[j] = row >= n ? 0.f : t < 0 ? NAN : a.coef ? a.coef[row] : 1.f;
        sub[j] = row < n ? a.lse[row] * LOG2E - 15.f : 0.f;   // P_SCALE = 2^15
        tgt[j] = t - pr.wm;
    }
    int nt = t0, nk = 0;
    auto next = [&](int buf) FA2_INLINE {
        if (nt >= t1) return false;
        pr.issue(nk, buf);
        nk += PK;
        if (nk == a.dp) {
            nk = 0;
            if (++nt < t1) pr.A.init(a.w, a.w_stride, a.p0 + nt * Pr::TM, a.V, a.wd);
        }
        return true;
    };
    typename Pr::Stream stream;
    pr.begin(stream, next);
    char *blk = out + (threadIdx.x >> 6) * 4096;
    for (int t = t0; t < t1; ++t) {
        const int v0 = a.p0 + t * Pr::TM;
        f16x acc[Pr::MI][Pr::NI];
        pr.steps(stream, a.dp / PK, acc, next);
#pragma unroll
        for (int j = 0; j < Pr::NI; ++j) {
            // rows of 64 elements in panel (row / 64, (t * TM + wm) / 64 + i / 2)
            const int row = rb * Pr::TN + pr.wn + 32 * j;
            T *o = static_cast<T *>(a.Pn) + ((int64_t)(row >> 6) * (a.piece / 64) + ((t * Pr::TM + pr.wm) >> 6)) * 4096 + (row & 63) * 64;
#pragma unroll
            for (int i = 0; i < Pr::MI; i += 2) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
#pragma unroll
                    for (int r = 0; r < 16; ++r) acc[i + h][j][r] = __builtin_amdgcn_exp2f(acc[i + h][j][r] * LOG2E - sub[j]);
                    const int at = tgt[j] - v0 - 32 * (i + h);
                    if (__any(at >= 0 && at < 32)) {
                        FA2_COLD_BRANCH();
#pragma unroll
                        for (int r = 0; r < 16; ++r)
                            if (at == acc_row(r, g2)) acc[i + h][j][r] -= P_SCALE;
                    }
                    if (v0 + pr.wm + 32 * (i + h) + 32 > a.V) {   // rows past the vocabulary
                        FA2_COLD_BRANCH();
#pragma unroll
                        for (int r = 0; r < 16; ++r)
                            if (v0 + pr.wm + 32 * (i + h) + acc_row(r, g2) >= a.V) acc[i + h][j][r] = 0.f;
                    }
                }
                store_rows<T>(acc[i][j], acc[i + 1][j], f[j], blk, o + (i / 2) * 4096, 64, 32, 64, true);
            }
        }
    }
}

// A tile of the piece's dW, or of a slice of its k: M side hidden columns, N side
// vocabulary rows, K packed tokens.
template <typename T, int MP>
__device__ __forceinline__ void xent_dw_item(const XentArgs &a, int item, int n, char *mem) {
    typedef Product<T, false, false, CLAMPED, PANELED, MP, MP, 2, 4> Pr;
    const int nd = (a.d + Pr::TM - 1) / Pr::TM, nv = (a.v1 - a.v0 + Pr::TM - 1) / Pr::TM;
    const int db = item % nd, vb = item / nd % nv, s = item / nd / nv;
    const int kt = (n + Pr::TM - 1) / Pr::TM * MP;
    const int k0 = (int)((int64_t)kt * s / a.wsplit) * PK, k1 = (int)((int64_t)kt * (s + 1) / a.wsplit) * PK;
    Pr pr;
    pr.init(mem);
    pr.A.init(a.xc, a.dp, db * Pr::TM, a.dp, a.rows_pad);
    pr.B.init(a.P, a.piece / 64, vb * Pr::TN);
    f16x acc[Pr::MI][Pr::NI];
    pr.run(k0, k1, acc);
    const int lane = threadIdx.x & 63, c = lane & 31, g2 = lane >> 5;
    const float u = xent_unscale(a, n);
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
template <typename T, Source W, int MP>
__device__ __forceinline__ void xent_dx_item(const XentArgs &a, const XentWork &k, int item, char *mem) {
    typedef Product<T, true, false, PANELED, W, MP, MP, 2, 4> Pr;
    const int nd = (a.d + Pr::TN - 1) / Pr::TN;
    const int db = item % nd, rb = item / nd % k.rt, s = item / nd / k.rt;
    const int kt = (a.v1 - a.v0 + PK - 1) / PK;
    const int k0 = (int)((int64_t)kt * s / k.xs) * PK, k1 = (int)((int64_t)kt * (s + 1) / k.xs) * PK;
    Pr pr;
    pr.init(mem);
    pr.A.init(a.P, a.piece / 64, rb * Pr::TM);
    pr.B.init(static_cast<const T *>(a.w) + (int64_t)a.v0 * a.w_stride, a.w_stride, db * Pr::TN, a.wd, a.V - a.v0);
    f16x acc[Pr::MI][Pr::NI];
    pr.run(k0, k1, acc);
    const int lane = threadIdx.x & 63, c = lane & 31, g2 = lane >> 5;
#pragma unroll
    for (int j = 0; j < Pr::NI; ++j) {
        const int col = db * Pr::TN + pr.wn + 32 * j + c;
        if (col >= a.dp) continue;
#pragma unroll
        for (int i = 0; i < Pr::MI; ++i) {
            float *o = a.acc + ((int64_t)(s * k.rt + rb) * Pr::TM + pr.wm + 32 * i) * a.dp + col;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                float *q = o + (int64_t)acc_row(r, g2) * a.dp;
                *q = a.v0 == 0 ? acc[i][j][r] : *q + acc[i][j][r];
            }
        }
    }
}

// MP = 4: 160 KB of LDS, one workgroup a compute unit; P's output goes through LDS of
// its own while the next tile's stages land.  MP = 2: 64 KB, two a unit, one tile of P
// an item, whose output goes through the panels.
//
// Bound by the matrix units and the board's power, and by units that idle at a launch's
// end: 16384 tokens x 8192 columns x 768, dW and dx of a piece beside P of the next,
// take 600 us, 1030 TFLOP/s; a last piece of 7424 columns without a P beside it 400 us,
// 930.  Pieces of half the size: the whole gradient 17% slower; of twice the size: 3%
// faster, for 1 GiB of scratch instead of 512 MiB.
template <typename T, Source W, int MP>
__global__ __launch_bounds__(512, 2) void xent_grad_kernel(const XentArgs a) {
    constexpr int PANELS = Product<T, true, true, W, PADDED, MP, MP, 2, 4>::LDS;
    __shared__ __align__(16) char mem[PANELS + (MP == 4 ? 8 * 4096 : 0)];
    const int n = a.count[N_TOKENS];
    const XentWork k = xent_work<MP>(a, n);
    int l = blockIdx.x;
    const bool dw_first = (int64_t)n * k.xs > (int64_t)(a.v1 - a.v0) * a.wsplit;   // the longer ones
    if (dw_first && l < k.dw) return xent_dw_item<T, MP>(a, xcd_item(l, k.dw), n, mem);
    l -= dw_first ? k.dw : 0;
    if (l < k.dx) return xent_dx_item<T, W, MP>(a, k, xcd_item(l, k.dx), mem);
    l -= k.dx;
    if (!dw_first && l < k.dw) return xent_dw_item<T, MP>(a, xcd_item(l, k.dw), n, mem);
    l -= dw_first ? 0 : k.dw;
    if (l < k.p) xent_p_item<T, W, MP>(a, k, xcd_item(l, k.p), n, mem, mem + (MP == 4 ? PANELS : 0));
}

// Eight elements of a row of `cols`, rounded; whole 16-byte stores where `vec`.
template <typename T>
__device__ __forceinline__ void store8(T *row, int c, int cols, bool vec, const f8 &x) {
    const typename vec_of<T>::v8 v = __builtin_convertvector(x, typename vec_of<T>::v8);
    if (vec) {
        *reinterpret_cast<typename vec_of<T>::v8 *>(row + c) = v;
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (c + e < cols) row[c + e] = v[e];
    }
}

// dW of a piece whose k was sliced: the slices' sums in order, one wave a row.
template <typename T>
__global__ __launch_bounds__(256) void xent_dw_join_kernel(const XentArgs a) {
    const float u = xent_unscale(a, a.count[N_TOKENS]);
    const int lane = threadIdx.x & 63;
    for (int v = blockIdx.x * 4 + (threadIdx.x >> 6); v < a.v1 - a.v0; v += gridDim.x * 4)
        for (int c = lane * 8; c < a.d; c += 512) {
            f8 x = {};
            for (int s = 0; s < a.wsplit; ++s) x += *reinterpret_cast<const f8 *>(a.wacc + ((int64_t)s * a.piece + v) * a.dp + c);
            store8<T>(static_cast<T *>(a.dw) + (int64_t)(a.v0 + v) * a.d, c, a.d, a.d % 8 == 0, x * u);
        }
}

// dx of every token: the slices' sums, rounded once; zeros where a token does not
// count.  One wave 256 columns of a token, eight slices' loads at a time (whole rows a
// wave, slice after slice: 38 us for 43 slices of 188 tokens).
template <typename T, int MP>
__global__ __launch_bounds__(256) void xent_dx_out_kernel(const XentArgs a) {
    const int n = a.count[N_TOKENS];
    const XentWork k = xent_work<MP>(a, n);
    const float u = xent_unscale(a, n);
    const int64_t slice = (int64_t)k.rt * (64 * MP) * a.dp;
    const int c = blockIdx.y * 256 + (threadIdx.x & 63) * 4;
    if (c >= a.d) return;
    for (int64_t i = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); i < a.rows; i += (int64_t)gridDim.x * 4) {
        const int j = a.pos[i];
        f4 x = {0.f, 0.f, 0.f, 0.f};
        if (j >= 0) {
            const float *p = a.acc + (int64_t)j * a.dp + c;
            int s = 0;
            for (; s + 8 <= k.xs; s += 8) {
                f4 v[8];
#pragma unroll
                for (int q = 0; q < 8; ++q) v[q] = *reinterpret_cast<const f4 *>(p + (s + q) * slice);
#pragma unroll
                for (int q = 0; q < 8; ++q) x += v[q];
            }
            for (; s < k.xs; ++s) x += *reinterpret_cast<const f4 *>(p + s * slice);
        }
        store4(static_cast<T *>(a.dx) + i * a.d, c, a.d, a.d % 4 == 0, x * u);
    }
}

#define FA2_LAUNCH(kernel, grid, block)                                    \
    do {                                                                   \
        hipLaunchKernelGGL(kernel, dim3(grid), dim3(block), 0, st, a);     \
        const hipError_t e = hipGetLastError();                            \
        if (e != hipSuccess) return e;                                     \
    } while (0)

// Hidden sizes that 64 does not divide have kernels of their own (W = RAGGED): the test
// for a stage's end costs the others 1% of the forward.  A padded copy of the weight
// instead: scoring of 130 tokens x 17428 x 1160 54 us, against 28.
unsigned at_most(int64_t want, int64_t most) { return (unsigned)(want < most ? want : most); }

template <typename T, Source W>
hipError_t fwd(const XentArgs &a, hipStream_t st) {
    if (!a.direct) FA2_LAUNCH(xent_pack_kernel<T>, at_most(a.rows_pad / a.pack_rows, 1024), 1024);
    if (a.stat_tile_n == 64)
        FA2_LAUNCH((xent_stats_kernel<T, W, 2, 1, 4, 2, 3>), a.stat_items, 512);
    else if (a.stat_tile_m == 128)
        FA2_LAUNCH((xent_stats_kernel<T, W, 2, 4, 2, 4, 3>), a.stat_items, 512);
    else
        FA2_LAUNCH((xent_stats_kernel<T, W, 4, 4, 2, 4, 2>), a.stat_items, 512);
    if (a.rows > 0) FA2_LAUNCH(xent_join_kernel<T>, (unsigned)((a.rows + 3) / 4), 256);
    if (a.reduction != FA2_REDUCE_NONE) FA2_LAUNCH(xent_sum_kernel, 1, 1024);
    return hipSuccess;
}

// P of [p0, p1) beside dW and dx of [v0, v1); either may be empty.
template <typename T, Source W, int MP>
hipError_t grad(const XentArgs &a, hipStream_t st) {
    const int nv = a.v1 - a.v0, items = xent_work_most<MP>(a);
    if (items > 0) FA2_LAUNCH((xent_grad_kernel<T, W, MP>), items, 512);
    if (nv && a.dw && a.wsplit > 1) FA2_LAUNCH(xent_dw_join_kernel<T>, at_most((nv + 3) / 4, 8192), 256);
    return hipSuccess;
}

template <typename T, Source W>
hipError_t grad_sized(const XentArgs &a, hipStream_t st) {
    return a.small ? grad<T, W, 2>(a, st) : grad<T, W, 4>(a, st);
}

}  // namespace

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
    if (a.wd % PK) return a.type == FA2_F16 ? fwd<_Float16, RAGGED>(a, st) : fwd<__bf16, RAGGED>(a, st);
    return a.type == FA2_F16 ? fwd<_Float16, CLAMPED>(a, st) : fwd<__bf16, CLAMPED>(a, st);
}

hipError_t launch_xent_bwd_prepare(const XentArgs &a, hipStream_t st) {
    FA2_LAUNCH(xent_coef_kernel, 1, 1024);
    return hipSuccess;
}

hipError_t launch_xent_grad(const XentArgs &a, hipStream_t st) {
    if (a.wd % PK) return a.type == FA2_F16 ? grad_sized<_Float16, RAGGED>(a, st) : grad_sized<__bf16, RAGGED>(a, st);
    return a.type == FA2_F16 ? grad_sized<_Float16, CLAMPED>(a, st) : grad_sized<__bf16, CLAMPED>(a, st);
}

hipError_t launch_xent_bwd_finish(const XentArgs &a, hipStream_t st) {
    const dim3 grid(at_most((a.rows + 3) / 4, 4096), (a.d + 255) / 256);
    if (a.type == FA2_F16) {
        if (a.small)
            FA2_LAUNCH((xent_dx_out_kernel<_Float16, 2>), grid, 256);
        else
            FA2_LAUNCH((xent_dx_out_kernel<_Float16, 4>), grid, 256);
    } else {
        if (a.small)
            FA2_LAUNCH((xent_dx_out_kernel<__bf16, 2>), grid, 256);
        else
            FA2_LAUNCH((xent_dx_out_kernel<__bf16, 4>), grid, 256);
    }
    return hipSuccess;
}

}  // namespace fa2
