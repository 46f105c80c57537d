// fa2_token.h -- argument blocks, launch entry points and device helpers of the
// operators that work on token rows [rows, cols]: RMS norm with the residual's
// addition (fa2_norm.hip), dropout (fa2_dropout.hip) and the language model
// head with its cross entropy (fa2_xent.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "../../include/fa2_mi355x.h"
#include "fa2_device.h"

namespace fa2 {

typedef __bf16 b2 __attribute__((ext_vector_type(2)));
typedef __bf16 b4 __attribute__((ext_vector_type(4)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));

template <typename T>
struct vec_of;
template <>
struct vec_of<_Float16> {
    typedef h4 v4;
    typedef h8 v8;
};
template <>
struct vec_of<__bf16> {
    typedef b4 v4;
    typedef b8 v8;
};
template <>
struct vec_of<float> {
    typedef f4 v4;
    typedef f8 v8;
};

struct NormFwdArgs {
    const void *x, *res, *w;     // res null: h = x
    void *h, *y;                 // h null: not stored
    float *rstd, *scale;         // rstd null: not stored; scale: 8-bit output only
    int64_t x_stride, res_stride;
    int64_t rows;
    int cols;
    float eps;
    int w_type;
    int vec;                     // every row of every tensor takes four-element loads
    uint32_t seed_part;          // dropout_row_part(seed, -1, 0): the hash's terms of seed and head
    uint32_t drop_thr;           // 0: no dropout
    float inv_keep;
    bool stream;                 // rows_stream of x and the residual
};

struct NormBwdArgs {
    const void *dy, *dh, *h, *w; // dh null: no gradient through h
    const float *rstd;
    void *dx, *dres;             // dres null: not wanted
    void *dw;                    // null: not wanted
    float *part;                 // [blocks, cols] partial sums of dw
    int64_t dy_stride, dh_stride, h_stride;
    int64_t rows;
    int cols;
    int w_type, dw_type;
    int vec;
    int blocks;
    uint32_t seed_part, drop_thr;
    float inv_keep;
    bool stream;                 // rows_stream of dy, h and dh
};

struct DropoutArgs {
    const void *x;
    void *y;
    int64_t x_stride, rows;
    int cols;
    int vec;
    uint32_t seed_part, drop_thr;
    float inv_keep;
};

// Language model head with cross entropy.  Token rows that count (target not
// ignore_index) are packed to the front: packed row j is token rowmap[j], rows
// are `rows_pad` (a multiple of XENT_PAD) with zeros behind the last one.
constexpr int XENT_PAD = 256;      // packed rows and a piece's columns: multiples of this
constexpr int XENT_KPAD = 64;      // the hidden size the products see: a multiple of this

// Slices of the vocabulary for the forward over n tokens: the workgroups (token tiles x
// slices) fill the slots once, or a few times where that leaves fewer of them idle; the
// cost of a choice is its rounds times the tiles of a slice.
__host__ __device__ inline int xent_stat_splits(int tile_n, int tile_m, int slots, int rounds, int n, int V) {
    const int rt = n > tile_n ? (n + tile_n - 1) / tile_n : 1, tiles = (V + tile_m - 1) / tile_m;
    int best = 1, cost = INT32_MAX;
    for (int k = 1; k <= rounds; ++k) {
        int s = k * slots / rt;
        s = s < 1 ? 1 : s > tiles ? tiles : s;
        const int c = (rt * s + slots - 1) / slots * ((tiles + s - 1) / s);
        if (c < cost) {
            cost = c;
            best = s;
        }
    }
    return best;
}

struct XentArgs {
    int64_t rows;                  // N
    int rows_pad;
    int d, dp;                     // hidden size; padded to XENT_KPAD
    int V;
    int type;
    const void *x;                 // [N, d]
    int64_t x_stride;
    const void *w;                 // [V, wd]: the weight, wd = d, or its padded copy, wd = dp
    int64_t w_stride;
    int wd;
    const int64_t *target;
    int64_t ignore;
    int reduction;
    // kept for the backward
    int *count;                    // tokens that count, slices of the forward
    int *pos;                      // [N]: packed row of a token, -1 where ignored
    int *rowmap;                   // [rows_pad]
    int *tgt;                      // [rows_pad]: target, -1 where it is outside the vocabulary
    float *lse;                    // [rows_pad]
    void *xc;                      // [rows_pad, dp]; direct: the states themselves
    int64_t xc_stride;
    // forward
    int pack_rows;                 // packed rows a workgroup has at a time
    bool direct;                   // nothing is packed: every token is a row, nothing is kept
    int stat_tile_n, stat_tile_m;  // tokens and vocabulary rows of a tile
    int stat_slots, stat_rounds;   // workgroups resident at once; rounds of them to consider
    int stat_splits;               // direct: slices of the vocabulary
    int stat_items;                // workgroups there are partial results for
    float *part;                   // [token][slice] (maximum, sum)
    float *row_loss;               // sum, mean: [N]
    float *loss;                   // scalar, or [N]
    // backward
    const float *g;                // gradient of loss
    int g_stride;                  // none: elements between rows of g
    float *coef;                   // none: [rows_pad] factor of a row of P; else null
    float *unscale;                // none: [1] factor of the finished products
    bool small;                    // tiles of 128, not 256
    int slots;                     // workgroups resident at once
    int piece, pieces;             // vocabulary columns of a piece; pieces
    int v0, v1;                    // the piece whose dW and dx are formed, from P
    const void *P;                 // [rows_pad / 64, piece / 64] panels of 64 x 64
    int p0, p1;                    // the piece whose P is formed, into Pn
    void *Pn;
    int xcap;                      // dx: token tiles there are sums for, in all slices
    float *acc;                    // [xcap tiles, dp]
    int wsplit;                    // dW: slices of the tokens
    float *wacc;                   // [wsplit, piece, dp]; only with slices
    void *dx, *dw;                 // [N, d], [V, d]; null: not wanted
};

// The work of one launch of the backward: dW and dx of a piece, and P of the piece
// after it, as items of one grid, the long ones first; P's many short items fill the
// compute units that the others leave.  Lengths are in stages of 64 k; tiles are
// 64 MP on a side.
struct XentWork {
    int rt;            // tiles of tokens that count
    int dw, dx, p;     // items
    int xs;            // slices of dx's k
    int strip;         // tiles of P an item
};

constexpr int P_ROUNDS = 4;         // items of P a slot, at most
constexpr int P_TILE_EXTRA = 4;     // stages that the softmax of a tile of P takes as long as

template <typename N>
__host__ __device__ inline N larger(N a, N b) {
    return a > b ? a : b;
}
template <typename N>
__host__ __device__ inline N smaller(N a, N b) {
    return a < b ? a : b;
}

template <int MP>
__host__ __device__ inline XentWork xent_work(const XentArgs &a, int n) {
    constexpr int TT = 64 * MP;
    XentWork k;
    const int nd = (a.d + TT - 1) / TT, nv = (a.v1 - a.v0 + TT - 1) / TT, nvp = (a.p1 - a.p0 + TT - 1) / TT;
    k.rt = (n + TT - 1) / TT;
    // Slices of dx: no longer than half a slot's share of a launch (with pieces of full
    // width; the same number for every piece).  Of 6353 tokens x 32003 x 512 forward and
    // backward: 903 us, with three quarters 912, with a third 964; 9696 x 24723 x 256:
    // 636, 646, 684; wider hidden sizes within 0.3%.
    const int64_t total = (int64_t)(a.piece / TT) * k.rt * (nd * 2 * MP + (a.pieces > 1 ? a.dp / XENT_KPAD + P_TILE_EXTRA : 0));
    const int share = (int)larger((int64_t)4, total / (2 * a.slots));
    k.xs = larger(1, smaller((a.piece / XENT_KPAD + share - 1) / share, a.xcap / larger(k.rt, 1)));
    k.dw = a.dw ? nd * nv * a.wsplit : 0;
    k.dx = a.dx && nv > 0 ? nd * k.rt * k.xs : 0;
    // P: tiles of one token tile in strips, whose stages are one stream (MP = 2: single
    // tiles, since their output goes through the panels).  Alone, in the rounds of equal
    // strips that take the fewest tiles one after the other; beside the others short
    // ones, up to four a slot.
    const int tiles = k.rt * nvp;
    k.strip = MP == 2 ? 1 : larger(1, (tiles + P_ROUNDS * a.slots - 1) / (P_ROUNDS * a.slots));
    if (MP == 4 && k.dw + k.dx == 0) {
        int cost = INT32_MAX;
        for (int r = 1; r <= P_ROUNDS; ++r) {
            const int s = larger(1, (tiles + r * a.slots - 1) / (r * a.slots));
            const int c = (k.rt * ((nvp + s - 1) / s) + a.slots - 1) / a.slots * (4 * s + 1);   // a strip's start: a quarter tile
            if (c < cost) {
                cost = c;
                k.strip = s;
            }
        }
    }
    k.p = k.rt * ((nvp + k.strip - 1) / k.strip);
    return k;
}

// The most items that xent_work can give, whatever number of tokens counts.
template <int MP>
inline int xent_work_most(const XentArgs &a) {
    constexpr int TT = 64 * MP;
    const int rt = a.rows_pad / TT, nd = (a.d + TT - 1) / TT, nv = (a.v1 - a.v0 + TT - 1) / TT, np = (a.p1 - a.p0 + TT - 1) / TT;
    const int strips = MP == 2 ? rt * np : smaller(rt * np, P_ROUNDS * a.slots + rt);
    return (a.dw ? nd * nv * a.wsplit : 0) + (a.dx && nv ? nd * a.xcap : 0) + strips;
}

hipError_t launch_xent_fwd(const XentArgs &a, hipStream_t st);
hipError_t launch_xent_pad_weight(const void *w, int64_t w_stride, void *out, int V, int d, int dp, int type, hipStream_t st);
hipError_t launch_xent_bwd_prepare(const XentArgs &a, hipStream_t st);
hipError_t launch_xent_grad(const XentArgs &a, hipStream_t st);
hipError_t launch_xent_bwd_finish(const XentArgs &a, hipStream_t st);

// Rows are read by nontemporal loads when they take more than 88 MiB together (RoPE's
// rule): they leave the caches to what is written, which is read next.  32768 x 768, fp16
// branch and fp32 residual, forward and backward: 138.6 -> 127.1 us; 4096 x 1024 in 8 bits,
// whose rows are still in the Infinity Cache: 12.0 -> 14.6.
inline bool rows_stream(int64_t bytes) { return bytes > (int64_t)88 << 20; }

hipError_t launch_norm_fwd(const NormFwdArgs &a, int x_type, int res_type, int y_type, hipStream_t st);
hipError_t launch_norm_bwd(const NormBwdArgs &a, int x_type, int h_type, int y_type, hipStream_t st);
int norm_bwd_blocks(int64_t rows, int cols);
hipError_t launch_dropout(const DropoutArgs &a, int type, hipStream_t st);

// v under dropout, for element (row, col): the attention's generator with head 0;
// `part_row` holds the hash's terms of the seed, the head and the row.  A dropped
// element is 0 whatever it was (inf and NaN too).
__device__ __forceinline__ float drop(float v, uint32_t part_row, int col, uint32_t thr, float inv_keep) {
    return dropout_keep_hashed(part_row ^ dropout_col_term(col), thr) ? v * inv_keep : 0.f;
}

// Four elements of a row from column col on, as fp32; zero past the row's end.  vec:
// rows and width are multiples of four elements; else whole groups of four are still
// one load, of a type aligned to its elements only (global memory takes it).
// STREAM: the whole loads are nontemporal.
template <typename T, bool STREAM = false>
__device__ __forceinline__ f4 load4(const T *row, int col, int cols, bool vec) {
    typedef typename vec_of<T>::v4 v4;
    typedef T u4 __attribute__((ext_vector_type(4), aligned(sizeof(T))));
    f4 r = {0.f, 0.f, 0.f, 0.f};
    if (vec) {
        const v4 *p = reinterpret_cast<const v4 *>(row + col);
        if (col < cols) r = __builtin_convertvector(STREAM ? __builtin_nontemporal_load(p) : *p, f4);
    } else if (col + 4 <= cols) {
        r = __builtin_convertvector((v4)*reinterpret_cast<const u4 *>(row + col), f4);
    } else {
#pragma unroll
        for (int j = 0; j < 3; ++j)
            if (col + j < cols) r[j] = (float)row[col + j];
    }
    return r;
}

template <typename T>
__device__ __forceinline__ void store4(T *row, int col, int cols, bool vec, f4 v) {
    typedef typename vec_of<T>::v4 v4;
    typedef T u4 __attribute__((ext_vector_type(4), aligned(sizeof(T))));
    const v4 q = __builtin_convertvector(v, v4);
    if (vec) {
        if (col < cols) *reinterpret_cast<v4 *>(row + col) = q;
    } else if (col + 4 <= cols) {
        *reinterpret_cast<u4 *>(row + col) = q;
    } else {
#pragma unroll
        for (int j = 0; j < 3; ++j)
            if (col + j < cols) row[col + j] = q[j];
    }
}

// The same with the element type as an argument (uniform).
__device__ __forceinline__ f4 load4_typed(const void *row, int type, int col, int cols, bool vec) {
    if (type == FA2_F16) return load4(static_cast<const _Float16 *>(row), col, cols, vec);
    if (type == FA2_BF16) return load4(static_cast<const __bf16 *>(row), col, cols, vec);
    return load4(static_cast<const float *>(row), col, cols, vec);
}

__device__ __forceinline__ void store1_typed(void *p, int type, int64_t i, float v) {
    if (type == FA2_F16)
        static_cast<_Float16 *>(p)[i] = (_Float16)v;
    else if (type == FA2_BF16)
        static_cast<__bf16 *>(p)[i] = (__bf16)v;
    else
        static_cast<float *>(p)[i] = v;
}

// Sum (or, MAX, the largest value, NaN first) over the G lanes that share a row;
// G = 64: one wave, otherwise a whole workgroup, through `red` (one float a wave).
template <int G, bool MAX>
__device__ __forceinline__ float row_reduce(float v, float *red) {
    auto join = [](float a, float b) FA2_INLINE { return MAX ? ((b > a || b != b) ? b : a) : a + b; };
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) v = join(v, __shfl_xor(v, o));
    if (G > 64) {
        __syncthreads();   // the previous use of red has been read
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
        __syncthreads();
        v = red[0];
#pragma unroll
        for (int i = 1; i < G / 64; ++i) v = join(v, red[i]);
    }
    return v;
}

// Norm kernels: calls f(G, NCH) with the lanes a row takes and the four-element pieces a lane.
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

}  // namespace fa2
