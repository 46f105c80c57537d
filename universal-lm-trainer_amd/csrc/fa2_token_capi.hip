// fa2_token_capi.hip -- the C ABI of the operators on token rows: argument
// validation, plans and workspaces, launches.  Allocates nothing, keeps nothing
// between calls, never synchronises.
#include <math.h>
#include <string.h>

#include "fa2_kernels.h"
#include "fa2_token.h"

namespace {

using fa2::clear_error;
using fa2::fail;

size_t type_size(int t) { return t == FA2_F32 ? 4 : t == FA2_E4M3 ? 1 : 2; }
bool aligned(const void *p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }

int check_rows(const char *op, int64_t rows, int32_t cols, int32_t most) {
    if (rows < 0 || rows > INT32_MAX) return fail(FA2_ERR_BAD_SHAPE, "%s: %lld rows outside 0 .. 2^31 - 1", op, (long long)rows);
    if (cols < 1 || cols > most) return fail(FA2_ERR_BAD_SHAPE, "%s: row length %d outside 1 .. %d", op, cols, most);
    return FA2_OK;
}

int check_type(const char *name, int t, int last) {
    return t < 0 || t > last ? fail(FA2_ERR_BAD_ARGUMENT, "%s type %d is not known here", name, t) : (int)FA2_OK;
}

// A tensor of rows: pointer, element alignment, stride.
int check_row_tensor(const char *name, const void *p, int type, int64_t stride) {
    if (!p) return fail(FA2_ERR_NULL_POINTER, "%s is NULL", name);
    if (!aligned(p, type_size(type))) return fail(FA2_ERR_MISALIGNED, "%s is not aligned to its elements", name);
    if (stride < 0 || stride > (int64_t)1 << 31) return fail(FA2_ERR_BAD_SHAPE, "%s row stride %lld outside 0 .. 2^31", name, (long long)stride);
    return FA2_OK;
}

// Whether rows of a tensor take loads of n elements.
bool vector_rows(const void *p, int type, int64_t stride, int n) {
    return !p || (aligned(p, n * type_size(type) < 16 ? n * type_size(type) : 16) && stride % n == 0);
}

int check_dropout(float p) {
    return p >= 0.f && p < 1.f ? (int)FA2_OK : fail(FA2_ERR_BAD_ARGUMENT, "dropout_p %g outside [0, 1)", (double)p);
}

// The hash's terms of the seed and of head 0 (dropout_row_part without its row).
uint32_t seed_part(uint32_t seed) { return (seed * 0x9E3779B1u) ^ 0x27D4EB2Fu; }

float inv_keep(float p) { return (float)(1.0 / (1.0 - (double)p)); }

int launched(const char *op, hipError_t e) {
    return e == hipSuccess ? (int)FA2_OK : fail(FA2_ERR_LAUNCH, "%s launch: %s", op, hipGetErrorString(e));
}

int check_norm_types(int x, int res, int y, bool fp8) {
    int rc;
    if ((rc = check_type("x", x, FA2_F32)) || (rc = check_type("residual", res, FA2_F32)) ||
        (rc = check_type("y", y, fp8 ? FA2_E4M3 : FA2_F32)))
        return rc;
    if (res != x && res != FA2_F32) return fail(FA2_ERR_BAD_ARGUMENT, "the residual must be of x's type or fp32");
    if (y != x && x != FA2_F32 && y != FA2_E4M3) return fail(FA2_ERR_BAD_ARGUMENT, "y must be of x's type");
    return FA2_OK;
}

// ---------------------------------------------------------------------------
// Cross entropy: sizes and buffers that follow from (rows, hidden, vocab).
// ---------------------------------------------------------------------------
struct XentPlan {
    int rows_pad, dp;
    bool small;
    int stat_tile_n, stat_tile_m, stat_slots, stat_rounds, stat_items;
    int slots, piece, pieces, xcap;
    int wsplit, wsplit_last;
    // offsets in the state
    size_t count, lse, tgt, rowmap, pos, xc, state_bytes;
    // offsets in the forward's workspace
    size_t f_weight, part, row_loss, fwd_bytes;
    // offsets in the backward's workspace
    size_t b_weight, coef, unscale, P[2], acc, wacc, bwd_bytes;
};

int64_t clamp(int64_t v, int64_t lo, int64_t hi) { return v < lo ? lo : v > hi ? hi : v; }

// Sizes that must not depend on how many tokens count, which only the device knows;
// the kernels choose the slices of the forward and of dx within them.
XentPlan xent_plan(int64_t rows, int32_t d, int32_t V) {
    using namespace fa2;
    XentPlan p;
    p.rows_pad = (int)((rows + XENT_PAD - 1) / XENT_PAD * XENT_PAD);
    p.dp = (d + XENT_KPAD - 1) / XENT_KPAD * XENT_KPAD;
    const int64_t R = p.rows_pad;
    // Forward: tiles of 256 tokens x 256 vocabulary rows, one workgroup a compute unit;
    // where those are fewer than two a unit, 256 x 128 (and a deeper stream of stages); up
    // to 64 tokens, and where even these leave half the units idle, 64 x 128, two a unit.
    const int64_t t256 = R / 256, v256 = (V + 255) / 256, v128 = (V + 127) / 128;
    p.stat_tile_m = t256 * v256 < 512 ? 128 : 256;
    p.stat_tile_n = p.stat_tile_m == 128 && (rows <= 64 || t256 * v128 < 128) ? 64 : 256;
    p.stat_slots = p.stat_tile_n == 64 ? 512 : 256;
    p.stat_rounds = p.stat_tile_m == 256 ? 4 : 2;
    const int64_t token_tiles = (rows + p.stat_tile_n - 1) / p.stat_tile_n, v_tiles = p.stat_tile_m == 256 ? v256 : v128;
    p.stat_items = (int)(token_tiles > p.stat_slots * p.stat_rounds ? token_tiles : p.stat_slots * p.stat_rounds);
    if (p.stat_items > token_tiles * v_tiles) p.stat_items = (int)(token_tiles * v_tiles);
    // Backward.  A piece's P is at most 256 MiB (twice, with more than one piece), or 256
    // columns from 2^19 tokens on, in equal pieces.
    const int64_t most = clamp(((int64_t)256 << 20) / (2 * R) / XENT_PAD * XENT_PAD, XENT_PAD, 1 << 24);
    p.pieces = (int)((V + most - 1) / most);
    p.piece = (int)(((V + p.pieces - 1) / p.pieces + XENT_PAD - 1) / XENT_PAD * XENT_PAD);
    p.pieces = (V + p.piece - 1) / p.piece;
    // Tiles of 128 where P has fewer tiles of 256 than there are compute units.
    p.small = (R / 256) * (p.piece / 256) < 256;
    p.slots = p.small ? 512 : 256;
    const int64_t tt = p.small ? 128 : 256, rt = R / tt, nd = (d + tt - 1) / tt, nv = p.piece / tt;
    // dx: sums for all token tiles, or, when those are few, for slices up to one item a slot.
    p.xcap = (int)(rt * nd > p.slots ? rt : clamp(p.slots / nd, 1, p.slots));
    // dW: its k, the tokens, in slices (lengths in stages of 64 k).  Beside P, whose items
    // fill the slots, none longer than a slot's share of the launch; without P, thirds of
    // a share where a whole one is longer than half of it.
    const int64_t kt = rt * (tt / 64), both = nv * rt * (nd * 2 * (tt / 64)) / p.slots, fill = nv * rt * (p.dp / 64 + 4) / p.slots;
    auto slices = [&](int64_t len) { return (int)clamp((kt + len - 1) / (len > 4 ? len : 4), 1, p.pieces > 1 ? 4 : 16); };
    p.wsplit = p.pieces > 1 ? slices(both + fill) : 1;
    p.wsplit_last = kt > both / 2 ? slices(both / 3) : 1;
    const int wmax = p.wsplit > p.wsplit_last ? p.wsplit : p.wsplit_last;
    size_t at = 0;
    auto take = [&](size_t bytes) { const size_t o = at; at += up256(bytes); return o; };
    p.count = take(256);
    p.lse = take(R * 4);
    p.tgt = take(R * 4);
    p.rowmap = take(R * 4);
    p.pos = take((size_t)rows * 4);
    p.xc = take((size_t)R * p.dp * 2);
    p.state_bytes = at;
    const size_t wbytes = d % 8 ? (size_t)V * p.dp * 2 : 0;
    at = 0;
    p.f_weight = take(wbytes);
    p.part = take((size_t)p.stat_items * p.stat_tile_n * 8);
    p.row_loss = take((size_t)rows * 4);
    p.fwd_bytes = at;
    at = 0;
    p.b_weight = take(wbytes);
    p.coef = take(R * 4);
    p.unscale = take(256);
    p.P[0] = take((size_t)R * p.piece * 2);
    p.P[1] = p.pieces > 1 ? take((size_t)R * p.piece * 2) : p.P[0];
    p.acc = take((size_t)p.xcap * tt * p.dp * 4);
    p.wacc = take(wmax > 1 ? (size_t)wmax * p.piece * p.dp * 4 : 0);
    p.bwd_bytes = at;
    return p;
}

bool xent_sizes_ok(int64_t rows, int32_t d, int32_t V) {
    return rows >= 0 && rows <= (1 << 24) && d >= 1 && d <= FA2_ROW_MAX && V >= 1 && V <= (1 << 24);
}

int xent_check(const fa2_xent_params *p, const void *ws, size_t ws_bytes, bool backward) {
    if (!p) return fail(FA2_ERR_NULL_POINTER, "params is NULL");
    if (!xent_sizes_ok(p->rows, p->hidden, p->vocab))
        return fail(FA2_ERR_BAD_SHAPE, "rows %lld, hidden %d, vocab %d outside 0 .. 2^24, 1 .. %d, 1 .. 2^24", (long long)p->rows,
                    p->hidden, p->vocab, FA2_ROW_MAX);
    int rc;
    if ((rc = check_type("x", p->type, FA2_BF16))) return rc;
    if (p->reduction < 0 || p->reduction > FA2_REDUCE_MEAN) return fail(FA2_ERR_BAD_ARGUMENT, "reduction %d is not known", p->reduction);
    if ((rc = check_row_tensor("weight", p->weight, p->type, p->weight_stride))) return rc;
    if (p->weight_stride >= 1 << 22) return fail(FA2_ERR_BAD_SHAPE, "weight row stride %lld is not below 2^22", (long long)p->weight_stride);
    if (p->weight_stride < p->hidden) return fail(FA2_ERR_BAD_SHAPE, "weight row stride %lld is below hidden", (long long)p->weight_stride);
    if (p->hidden % 8 == 0 && (!aligned(p->weight, 16) || p->weight_stride % 8))
        return fail(FA2_ERR_MISALIGNED, "weight needs a 16-byte aligned base and a row stride that is a multiple of 8");
    if (p->rows > 0) {
        if (!backward && (rc = check_row_tensor("x", p->x, p->type, p->x_stride))) return rc;
        if (!backward && !p->target) return fail(FA2_ERR_NULL_POINTER, "target is NULL");
        if (!backward && !aligned(p->target, 8)) return fail(FA2_ERR_MISALIGNED, "target is not 8-byte aligned");
    }
    const size_t state = fa2_xent_state_bytes(p->rows, p->hidden);
    const bool keeps = backward || p->state;
    if (keeps && (!p->state || p->state_bytes < state))
        return fail(FA2_ERR_WORKSPACE, "state needs %zu bytes, got %zu", state, p->state ? p->state_bytes : 0);
    const size_t need = backward ? fa2_xent_bwd_workspace_bytes(p->rows, p->hidden, p->vocab)
                                 : fa2_xent_fwd_workspace_bytes(p->rows, p->hidden, p->vocab) + (keeps ? 0 : state);
    if (!ws || ws_bytes < need) return fail(FA2_ERR_WORKSPACE, "workspace needs %zu bytes, got %zu", need, ws ? ws_bytes : 0);
    if (!aligned(ws, 16) || !aligned(p->state, 16)) return fail(FA2_ERR_MISALIGNED, "state and workspace must be 16-byte aligned");
    return FA2_OK;
}

fa2::XentArgs xent_args(const fa2_xent_params *p, const XentPlan &pl, char *s) {
    fa2::XentArgs a;
    memset(&a, 0, sizeof(a));
    a.rows = p->rows;
    a.rows_pad = pl.rows_pad;
    a.d = p->hidden;
    a.dp = pl.dp;
    a.V = p->vocab;
    a.type = p->type;
    a.x = p->x;
    a.x_stride = p->x_stride;
    a.w = p->weight;
    a.w_stride = p->weight_stride;
    a.wd = p->hidden;
    a.target = p->target;
    a.ignore = p->ignore_index;
    a.reduction = p->reduction;
    a.count = reinterpret_cast<int *>(s + pl.count);
    a.lse = reinterpret_cast<float *>(s + pl.lse);
    a.tgt = reinterpret_cast<int *>(s + pl.tgt);
    a.rowmap = reinterpret_cast<int *>(s + pl.rowmap);
    a.pos = reinterpret_cast<int *>(s + pl.pos);
    a.xc = s + pl.xc;
    a.xc_stride = pl.dp;
    a.pack_rows = pl.rows_pad <= 4096 ? 16 : 64;
    a.stat_tile_n = pl.stat_tile_n;
    a.stat_tile_m = pl.stat_tile_m;
    a.stat_slots = pl.stat_slots;
    a.stat_rounds = pl.stat_rounds;
    a.stat_items = pl.stat_items;
    a.small = pl.small;
    a.slots = pl.slots;
    a.piece = pl.piece;
    a.pieces = pl.pieces;
    a.xcap = pl.xcap;
    return a;
}

}  // namespace

extern "C" {

int fa2_rms_norm_fwd(const fa2_rms_norm_params *p, void *stream) {
    clear_error();
    if (!p) return fail(FA2_ERR_NULL_POINTER, "params is NULL");
    int rc = check_rows("rms_norm", p->rows, p->cols, FA2_ROW_MAX);
    if (rc) return rc;
    const int rtype = p->residual ? p->residual_type : p->x_type;
    if ((rc = check_norm_types(p->x_type, rtype, p->y_type, true)) || (rc = check_type("weight", p->weight_type, FA2_F32))) return rc;
    if ((rc = check_dropout(p->dropout_p))) return rc;
    if (p->dropout_p > 0.f && !p->residual) return fail(FA2_ERR_BAD_ARGUMENT, "dropout needs a residual to add to");
    if (!(p->eps >= 0.f) || !isfinite(p->eps)) return fail(FA2_ERR_BAD_ARGUMENT, "eps %g is negative or not finite", (double)p->eps);
    if (p->rows == 0) return FA2_OK;
    if ((rc = check_row_tensor("x", p->x, p->x_type, p->x_stride))) return rc;
    if ((rc = check_row_tensor("weight", p->weight, p->weight_type, 0))) return rc;
    if ((rc = check_row_tensor("y", p->y, p->y_type, 0))) return rc;
    if (p->residual) {
        if ((rc = check_row_tensor("residual", p->residual, rtype, p->residual_stride))) return rc;
        if ((rc = check_row_tensor("h", p->h, rtype, 0))) return rc;
    } else if (p->h) {
        return fail(FA2_ERR_BAD_ARGUMENT, "h is x without a residual: pass NULL");
    }
    if (p->y_type == FA2_E4M3 && !p->scale) return fail(FA2_ERR_NULL_POINTER, "scale is NULL");
    if (!aligned(p->rstd, 4) || !aligned(p->scale, 4)) return fail(FA2_ERR_MISALIGNED, "rstd / scale are not 4-byte aligned");
    fa2::NormFwdArgs a;
    a.x = p->x; a.res = p->residual; a.w = p->weight;
    a.h = p->h; a.y = p->y;
    a.rstd = p->rstd; a.scale = p->scale;
    a.x_stride = p->x_stride; a.res_stride = p->residual_stride;
    a.rows = p->rows; a.cols = p->cols;
    a.eps = p->eps;
    a.w_type = p->weight_type;
    a.vec = p->cols % 4 == 0 && vector_rows(p->x, p->x_type, p->x_stride, 4) &&
            vector_rows(p->residual, rtype, p->residual_stride, 4) && vector_rows(p->weight, p->weight_type, 0, 4) &&
            vector_rows(p->h, rtype, 0, 4) && vector_rows(p->y, p->y_type, 0, 4);
    a.seed_part = seed_part(p->seed);
    a.drop_thr = fa2_dropout_threshold(p->dropout_p);
    a.inv_keep = inv_keep(p->dropout_p);
    a.stream = fa2::rows_stream(p->rows * p->cols * (int64_t)(type_size(p->x_type) + (p->residual ? type_size(rtype) : 0)));
    return launched("rms_norm", fa2::launch_norm_fwd(a, p->x_type, rtype, p->y_type, (hipStream_t)stream));
}

size_t fa2_rms_norm_bwd_workspace_bytes(int64_t rows, int32_t cols) {
    if (rows <= 0 || cols <= 0) return 0;
    return up256((size_t)fa2::norm_bwd_blocks(rows, cols) * cols * sizeof(float));
}

int fa2_rms_norm_bwd(const fa2_rms_norm_bwd_params *p, void *workspace, size_t workspace_bytes, void *stream) {
    clear_error();
    if (!p) return fail(FA2_ERR_NULL_POINTER, "params is NULL");
    int rc = check_rows("rms_norm backward", p->rows, p->cols, FA2_ROW_MAX);
    if (rc) return rc;
    if ((rc = check_norm_types(p->x_type, p->h_type, p->y_type, false)) || (rc = check_type("weight", p->weight_type, FA2_F32))) return rc;
    if ((rc = check_dropout(p->dropout_p))) return rc;
    if (p->rows == 0 && !p->dweight) return FA2_OK;
    if (p->dweight && (rc = check_row_tensor("dweight", p->dweight, p->weight_type, 0))) return rc;
    if ((rc = check_row_tensor("weight", p->weight, p->weight_type, 0))) return rc;
    if (p->rows > 0) {
        if ((rc = check_row_tensor("dy", p->dy, p->y_type, p->dy_stride))) return rc;
        if ((rc = check_row_tensor("h", p->h, p->h_type, p->h_stride))) return rc;
        if (p->dh && (rc = check_row_tensor("dh", p->dh, p->h_type, p->dh_stride))) return rc;
        if (p->dx && (rc = check_row_tensor("dx", p->dx, p->x_type, 0))) return rc;
        if (p->dresidual && (rc = check_row_tensor("dresidual", p->dresidual, p->h_type, 0))) return rc;
        if (!p->rstd) return fail(FA2_ERR_NULL_POINTER, "rstd is NULL");
        if (!aligned(p->rstd, 4)) return fail(FA2_ERR_MISALIGNED, "rstd is not 4-byte aligned");
    }
    const size_t need = p->dweight ? fa2_rms_norm_bwd_workspace_bytes(p->rows, p->cols) : 0;
    if (need && (!workspace || workspace_bytes < need))
        return fail(FA2_ERR_WORKSPACE, "workspace needs %zu bytes, got %zu", need, workspace ? workspace_bytes : 0);
    if (need && !aligned(workspace, 16)) return fail(FA2_ERR_MISALIGNED, "workspace is not 16-byte aligned");
    fa2::NormBwdArgs a;
    a.dy = p->dy; a.dh = p->dh; a.h = p->h; a.w = p->weight;
    a.rstd = p->rstd;
    a.dx = p->dx; a.dres = p->dresidual; a.dw = p->dweight;
    a.part = static_cast<float *>(workspace);
    a.dy_stride = p->dy_stride; a.dh_stride = p->dh_stride; a.h_stride = p->h_stride;
    a.rows = p->rows; a.cols = p->cols;
    a.w_type = p->weight_type; a.dw_type = p->weight_type;
    a.vec = p->cols % 4 == 0 && vector_rows(p->dy, p->y_type, p->dy_stride, 4) && vector_rows(p->dh, p->h_type, p->dh_stride, 4) &&
            vector_rows(p->h, p->h_type, p->h_stride, 4) && vector_rows(p->weight, p->weight_type, 0, 4) &&
            vector_rows(p->dx, p->x_type, 0, 4) && vector_rows(p->dresidual, p->h_type, 0, 4);
    a.blocks = p->rows > 0 ? fa2::norm_bwd_blocks(p->rows, p->cols) : 0;
    a.seed_part = seed_part(p->seed);
    a.drop_thr = fa2_dropout_threshold(p->dropout_p);
    a.inv_keep = inv_keep(p->dropout_p);
    a.stream = fa2::rows_stream(p->rows * p->cols * (int64_t)(type_size(p->y_type) + type_size(p->h_type) * (p->dh ? 2 : 1)));
    return launched("rms_norm backward", fa2::launch_norm_bwd(a, p->x_type, p->h_type, p->y_type, (hipStream_t)stream));
}

int fa2_dropout(const fa2_dropout_params *p, void *stream) {
    clear_error();
    if (!p) return fail(FA2_ERR_NULL_POINTER, "params is NULL");
    int rc = check_rows("dropout", p->rows, p->cols, INT32_MAX);
    if (rc) return rc;
    if ((rc = check_type("x", p->type, FA2_F32)) || (rc = check_dropout(p->dropout_p))) return rc;
    if (p->rows == 0) return FA2_OK;
    if ((rc = check_row_tensor("x", p->x, p->type, p->x_stride)) || (rc = check_row_tensor("y", p->y, p->type, 0))) return rc;
    fa2::DropoutArgs a;
    a.x = p->x; a.y = p->y;
    a.x_stride = p->x_stride;
    a.rows = p->rows; a.cols = p->cols;
    a.vec = p->cols % 8 == 0 && vector_rows(p->x, p->type, p->x_stride, 8) && vector_rows(p->y, p->type, 0, 8);
    a.seed_part = seed_part(p->seed);
    a.drop_thr = fa2_dropout_threshold(p->dropout_p);
    a.inv_keep = inv_keep(p->dropout_p);
    return launched("dropout", fa2::launch_dropout(a, p->type, (hipStream_t)stream));
}

size_t fa2_xent_state_bytes(int64_t rows, int32_t hidden) {
    return xent_sizes_ok(rows, hidden, 1) ? xent_plan(rows > 0 ? rows : 1, hidden, 1).state_bytes : 0;
}
size_t fa2_xent_fwd_workspace_bytes(int64_t rows, int32_t hidden, int32_t vocab) {
    return xent_sizes_ok(rows, hidden, vocab) ? xent_plan(rows > 0 ? rows : 1, hidden, vocab).fwd_bytes : 0;
}
size_t fa2_xent_bwd_workspace_bytes(int64_t rows, int32_t hidden, int32_t vocab) {
    return xent_sizes_ok(rows, hidden, vocab) ? xent_plan(rows > 0 ? rows : 1, hidden, vocab).bwd_bytes : 0;
}

int fa2_xent_fwd(const fa2_xent_params *p, void *workspace, size_t workspace_bytes, void *stream) {
    clear_error();
    int rc = xent_check(p, workspace, workspace_bytes, false);
    if (rc) return rc;
    if (!p->loss && !(p->rows == 0 && p->reduction == FA2_REDUCE_NONE)) return fail(FA2_ERR_NULL_POINTER, "loss is NULL");
    if (!aligned(p->loss, 4)) return fail(FA2_ERR_MISALIGNED, "loss is not 4-byte aligned");
    const XentPlan pl = xent_plan(p->rows > 0 ? p->rows : 1, p->hidden, p->vocab);
    char *w = static_cast<char *>(workspace);
    fa2::XentArgs a = xent_args(p, pl, p->state ? static_cast<char *>(p->state) : w + pl.fwd_bytes);
    const hipStream_t st = (hipStream_t)stream;
    // Nothing kept, and states that the products can read: few enough tokens are not
    // packed (the weights' bytes, not the tokens, set the time), which saves a launch.
    a.direct = !p->state && p->reduction == FA2_REDUCE_NONE && pl.stat_tile_m == 128 && p->rows > 0 &&
               p->hidden % 8 == 0 && aligned(p->x, 16) && p->x_stride % 8 == 0 && p->x_stride < 1 << 22;
    if (a.direct) {
        a.xc = const_cast<void *>(p->x);
        a.xc_stride = p->x_stride;
        a.stat_splits = fa2::xent_stat_splits(a.stat_tile_n, a.stat_tile_m, a.stat_slots, a.stat_rounds, (int)p->rows, a.V);
    }
    a.part = reinterpret_cast<float *>(w + pl.part);
    a.row_loss = reinterpret_cast<float *>(w + pl.row_loss);
    a.loss = p->loss;
    hipError_t e = hipSuccess;
    if (p->hidden % 8) {
        e = fa2::launch_xent_pad_weight(p->weight, p->weight_stride, w + pl.f_weight, a.V, a.d, a.dp, a.type, st);
        a.w = w + pl.f_weight;
        a.w_stride = a.wd = a.dp;
    }
    if (e == hipSuccess) e = fa2::launch_xent_fwd(a, st);
    return launched("cross entropy", e);
}

int fa2_xent_bwd(const fa2_xent_params *p, void *workspace, size_t workspace_bytes, void *stream) {
    clear_error();
    int rc = xent_check(p, workspace, workspace_bytes, true);
    if (rc) return rc;
    if (!p->dx && !p->dweight) return FA2_OK;
    if (p->rows > 0 || p->reduction != FA2_REDUCE_NONE) {
        if (!p->dloss) return fail(FA2_ERR_NULL_POINTER, "dloss is NULL");
        if (!aligned(p->dloss, 4)) return fail(FA2_ERR_MISALIGNED, "dloss is not 4-byte aligned");
    }
    if (p->dloss_stride < 0 || p->dloss_stride > INT32_MAX) return fail(FA2_ERR_BAD_SHAPE, "dloss stride %lld outside 0 .. 2^31 - 1", (long long)p->dloss_stride);
    if (!aligned(p->dx, 16) || !aligned(p->dweight, 16)) return fail(FA2_ERR_MISALIGNED, "dx and dweight must be 16-byte aligned");
    const XentPlan pl = xent_plan(p->rows > 0 ? p->rows : 1, p->hidden, p->vocab);
    fa2::XentArgs a = xent_args(p, pl, static_cast<char *>(p->state));
    char *w = static_cast<char *>(workspace);
    const hipStream_t st = (hipStream_t)stream;
    a.g = p->dloss;
    a.g_stride = (int)p->dloss_stride;
    const bool per_row = p->reduction == FA2_REDUCE_NONE;
    a.coef = per_row ? reinterpret_cast<float *>(w + pl.coef) : nullptr;
    a.unscale = per_row ? reinterpret_cast<float *>(w + pl.unscale) : nullptr;
    a.acc = reinterpret_cast<float *>(w + pl.acc);
    a.wacc = reinterpret_cast<float *>(w + pl.wacc);
    a.dx = p->rows > 0 ? p->dx : nullptr;
    a.dw = p->dweight;
    hipError_t e = hipSuccess;
    if (p->hidden % 8) {
        e = fa2::launch_xent_pad_weight(p->weight, p->weight_stride, w + pl.b_weight, a.V, a.d, a.dp, a.type, st);
        a.w = w + pl.b_weight;
        a.w_stride = a.wd = a.dp;
    }
    if (e == hipSuccess && per_row) e = fa2::launch_xent_bwd_prepare(a, st);
    for (int i = 0; i <= a.pieces && e == hipSuccess; ++i) {   // P of piece i beside the gradients of piece i - 1
        auto edge = [&](int k) { return (int64_t)k * a.piece < a.V ? k * a.piece : a.V; };
        a.v0 = i > 0 ? edge(i - 1) : 0;
        a.v1 = i > 0 ? edge(i) : 0;
        a.p0 = edge(i);
        a.p1 = edge(i + 1);
        a.P = w + pl.P[(i + 1) & 1];
        a.Pn = w + pl.P[i & 1];
        a.wsplit = i == a.pieces ? pl.wsplit_last : pl.wsplit;
        e = fa2::launch_xent_grad(a, st);
    }
    if (e == hipSuccess && a.dx) e = fa2::launch_xent_bwd_finish(a, st);
    return launched("cross entropy backward", e);
}

}  // extern "C"
