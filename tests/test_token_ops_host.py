"""Operators on token rows, without a GPU: refusals of the C ABI (before any launch)
and of the Python entry points, workspace sizes, and the binding's ops."""
import ctypes

import pytest
import torch

import fa2_capi as capi
import flash_attn_v100_cuda as fa

BASE = 1 << 20   # never dereferenced: every call fails validation first


def _norm(**kw):
    p = capi.RmsNormParams()
    p.x = p.residual = p.weight = p.h = p.y = p.rstd = p.scale = BASE
    p.x_stride = p.residual_stride = 64
    p.rows, p.cols = 5, 64
    p.x_type, p.residual_type, p.weight_type, p.y_type = capi.F16, capi.F32, capi.F32, capi.F16
    p.eps, p.dropout_p, p.seed = 1e-6, 0.0, 0
    for k, v in kw.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("kw,status", [
    (dict(x=0), 1), (dict(weight=0), 1), (dict(y=0), 1), (dict(h=0), 1), (dict(y_type=capi.E4M3, scale=0), 1),
    (dict(rows=-1), 2), (dict(rows=1 << 31), 2), (dict(cols=0), 2), (dict(cols=8193), 2), (dict(x_stride=-1), 2),
    (dict(x=BASE + 1), 3), (dict(residual=BASE + 2), 3), (dict(rstd=BASE + 2), 3),
    (dict(x_type=7), 4), (dict(x_type=capi.E4M3), 4), (dict(residual_type=capi.BF16), 4), (dict(y_type=capi.F32), 4),
    (dict(dropout_p=1.0), 4), (dict(dropout_p=float("nan")), 4), (dict(eps=-1.0), 4), (dict(eps=float("inf")), 4),
    (dict(residual=0), 4),                                       # h without a residual
    (dict(residual=0, h=0, dropout_p=0.1), 4),                   # dropout without a residual
])
def test_norm_refusals(kw, status):
    lib = capi.load()
    rc = lib.fa2_rms_norm_fwd(ctypes.byref(_norm(**kw)), None)
    assert rc == status, (kw, rc, lib.fa2_last_error())
    assert lib.fa2_last_error() != b""


def _norm_bwd(**kw):
    p = capi.RmsNormBwdParams()
    p.dy = p.dh = p.h = p.weight = p.rstd = p.dx = p.dresidual = p.dweight = BASE
    p.dy_stride = p.dh_stride = p.h_stride = 64
    p.rows, p.cols = 5, 64
    p.x_type, p.h_type, p.weight_type, p.y_type = capi.F16, capi.F32, capi.F32, capi.F16
    for k, v in kw.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("kw,ws,status", [
    (dict(dy=0), 1 << 20, 1), (dict(h=0), 1 << 20, 1), (dict(rstd=0), 1 << 20, 1), (dict(cols=20000), 1 << 20, 2),
    (dict(dx=BASE + 1), 1 << 20, 3), (dict(y_type=capi.E4M3), 1 << 20, 4), (dict(dropout_p=-0.5), 1 << 20, 4),
    (dict(), 0, 5), (dict(), 4, 5)])
def test_norm_backward_refusals(kw, ws, status):
    lib = capi.load()
    rc = lib.fa2_rms_norm_bwd(ctypes.byref(_norm_bwd(**kw)), BASE if ws else None, ws, None)
    assert rc == status, (kw, rc, lib.fa2_last_error())


def test_norm_workspace_bytes():
    lib = capi.load()
    assert lib.fa2_rms_norm_bwd_workspace_bytes(0, 768) == 0
    assert lib.fa2_rms_norm_bwd_workspace_bytes(1, 64) >= 64 * 4
    assert lib.fa2_rms_norm_bwd_workspace_bytes(1 << 30, 8192) <= 1 << 26


@pytest.mark.parametrize("kw,status", [(dict(x=0), 1), (dict(y=0), 1), (dict(rows=1 << 31), 2), (dict(cols=0), 2),
                                       (dict(x=BASE + 1), 3), (dict(type=capi.E4M3), 4), (dict(dropout_p=1.0), 4)])
def test_dropout_refusals(kw, status):
    lib = capi.load()
    p = capi.DropoutParams()
    p.x = p.y = BASE
    p.x_stride, p.rows, p.cols, p.type, p.dropout_p = 64, 3, 64, capi.F16, 0.1
    for k, v in kw.items():
        setattr(p, k, v)
    assert lib.fa2_dropout(ctypes.byref(p), None) == status, lib.fa2_last_error()


def _xent(lib, **kw):
    p = capi.XentParams()
    p.x = p.weight = p.target = p.loss = p.state = p.dloss = p.dx = p.dweight = BASE
    p.x_stride = p.weight_stride = p.hidden = 128
    p.rows, p.vocab = 10, 100
    p.type, p.reduction, p.ignore_index = capi.F16, 2, -100
    p.state_bytes = lib.fa2_xent_state_bytes(10, 128)
    for k, v in kw.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("kw,status", [
    (dict(x=0), 1), (dict(weight=0), 1), (dict(target=0), 1), (dict(loss=0), 1),
    (dict(rows=(1 << 24) + 1), 2), (dict(hidden=0), 2), (dict(hidden=20000), 2), (dict(vocab=0), 2),
    (dict(weight_stride=64), 2), (dict(weight=BASE + 8), 3), (dict(weight_stride=132), 3), (dict(target=BASE + 4), 3),
    (dict(type=capi.F32), 4), (dict(reduction=3), 4), (dict(state_bytes=100), 5),
    (dict(state=0), 5)])   # without a state the workspace holds it too
def test_cross_entropy_refusals(kw, status):
    lib = capi.load()
    ws = lib.fa2_xent_fwd_workspace_bytes(10, 128, 100)
    p = _xent(lib, **kw)
    assert lib.fa2_xent_fwd(ctypes.byref(p), BASE, ws, None) == status, lib.fa2_last_error()


def test_cross_entropy_workspace_refusals():
    lib = capi.load()
    p = _xent(lib)
    assert lib.fa2_xent_fwd(ctypes.byref(p), BASE, lib.fa2_xent_fwd_workspace_bytes(10, 128, 100) - 1, None) == 5
    need = lib.fa2_xent_bwd_workspace_bytes(10, 128, 100)
    assert lib.fa2_xent_bwd(ctypes.byref(p), BASE, need - 1, None) == 5
    assert lib.fa2_xent_bwd(ctypes.byref(p), None, need, None) == 5
    assert lib.fa2_xent_bwd(ctypes.byref(p), BASE + 8, need, None) == 3
    p.dloss = 0
    assert lib.fa2_xent_bwd(ctypes.byref(p), BASE, need, None) == 1
    p.dx = p.dweight = 0   # nothing wanted: nothing to do
    assert lib.fa2_xent_bwd(ctypes.byref(p), BASE, need, None) == 0


@pytest.mark.parametrize("rows,d,V", [(0, 64, 10), (1, 1, 1), (16384, 768, 32000), (1 << 20, 768, 32000),
                                      (1 << 24, 64, 1 << 24), (37, 100, 50257)])
def test_cross_entropy_memory_is_bounded(rows, d, V):
    """Working memory next to the operands' own: one piece of the vocabulary, never [rows, V]."""
    lib = capi.load()
    pad = max(256, (rows + 255) // 256 * 256)
    dp = (d + 63) // 64 * 64
    copy = V * dp * 2 if d % 8 else 0
    assert lib.fa2_xent_state_bytes(rows, d) <= pad * (dp * 2 + 16) + rows * 4 + 4096
    # partial results of at most 1024 workgroups of 256 tokens, or one a token
    assert lib.fa2_xent_fwd_workspace_bytes(rows, d, V) <= copy + 8 * max(1024 * 256, pad) + 8 * pad + 8192
    # two pieces of at most 256 MiB (or of their least width, 256 columns), fp32 sums of dx for every token or
    # one item a slot, and of at most 16 slices of dW where tokens are many and the vocabulary is small
    piece = 2 * (max(256 << 20, pad * 512) + 512 * pad)
    slices = 4 * max(pad, 256 * 256) * dp + 16 * 4 * dp * min((V + 255) // 256 * 256, max(256, (256 << 20) // (2 * pad) + 256))
    assert lib.fa2_xent_bwd_workspace_bytes(rows, d, V) <= copy + piece + 4 * pad + slices + 8192


def test_module_surface():
    for name in ("rms_norm", "add_rms_norm", "rms_norm_fp8", "dropout", "linear_cross_entropy"):
        assert callable(getattr(fa, name))
    ext = fa.extension()
    for op in ("rms_norm", "add_rms_norm", "rms_norm_fp8", "dropout", "linear_cross_entropy"):
        assert hasattr(ext, op)


def test_cpu_tensors_are_refused():
    x, w, t = torch.zeros(3, 8), torch.zeros(8), torch.zeros(3, dtype=torch.long)
    for call in (lambda: fa.rms_norm(x, w), lambda: fa.add_rms_norm(x, x, w), lambda: fa.rms_norm_fp8(x, w),
                 lambda: fa.dropout(x, 0.1), lambda: fa.linear_cross_entropy(x.half(), torch.zeros(5, 8).half(), t)):
        with pytest.raises(ValueError):
            call()


def test_plans_stay_inside_their_buffers(tmp_path):
    """The slices that the kernels choose from the number of tokens that count fit the grids and buffers that the host sized
    without knowing it, over many sizes: forward slices, dx slices, items of every backward launch."""
    import os
    import subprocess
    csrc = os.path.join(capi.PKG, "csrc")
    src = tmp_path / "plans.cpp"
    src.write_text('#include "%s/fa2_token_capi.hip"\n' % csrc + r"""
#include <cstdio>
#include <cstdlib>
using namespace fa2;
template <int MP> static int check(XentArgs a, int n) {
    constexpr int TT = 64 * MP;
    const XentWork k = xent_work<MP>(a, n);
    const int nvp = (a.p1 - a.p0 + TT - 1) / TT;
    if (k.rt != (n + TT - 1) / TT || k.xs < 1 || k.strip < 1) return 1;
    if ((int64_t)k.xs * k.rt > a.xcap) return 2;
    if ((int64_t)k.dw + k.dx + k.p > xent_work_most<MP>(a)) return 3;
    if (MP == 2 && k.strip != 1) return 4;
    if ((int64_t)k.p * k.strip < (int64_t)k.rt * nvp) return 5;
    if (k.rt * TT > a.rows_pad) return 6;
    return 0;
}
int main() {
    srand(1);
    auto lo = [](double most) { double u = rand() / (RAND_MAX + 1.0); return (int64_t)exp(u * log(most)); };
    for (int it = 0; it < 200000; ++it) {
        const int64_t rows = lo(it % 3 ? 40000 : 16777217);
        const int d = (int)lo(8193), V = (int)lo(it % 5 ? 300000 : 16777217);
        const XentPlan p = xent_plan(rows, d, V);
        fa2_xent_params q;
        memset(&q, 0, sizeof(q));
        q.rows = rows; q.hidden = d; q.vocab = V;
        XentArgs a = xent_args(&q, p, nullptr);
        a.dw = a.dx = (void *)16;
        const int n = (int)(it % 4 == 0 ? rows : lo((double)rows + 1) - (it % 7 == 0));
        const int s = xent_stat_splits(a.stat_tile_n, a.stat_tile_m, a.stat_slots, a.stat_rounds, n, V);
        const int rt = n > 0 ? (n + a.stat_tile_n - 1) / a.stat_tile_n : 0;
        int bad = 0;
        if (s < 1 || (int64_t)rt * s > a.stat_items) bad = 10;
        if (s > (V + a.stat_tile_m - 1) / a.stat_tile_m) bad = 11;
        if (a.stat_items > (1 << 22)) bad = 12;                       // 2^22 workgroups of 512 threads
        for (int i = 0; i <= a.pieces && !bad; ++i) {
            auto edge = [&](int k) { return (int64_t)k * a.piece < V ? k * a.piece : V; };
            a.v0 = i ? edge(i - 1) : 0; a.v1 = i ? edge(i) : 0; a.p0 = edge(i); a.p1 = edge(i + 1);
            a.wsplit = i == a.pieces ? p.wsplit_last : p.wsplit;
            if (a.wsplit < 1 || a.wsplit > 16 || (i && a.v1 <= a.v0)) bad = 13;
            if (!bad) bad = a.small ? check<2>(a, n) : check<4>(a, n);
            if (i > 3 && i < a.pieces - 2) i = a.pieces - 3;
        }
        if (a.piece % 256 || (int64_t)a.pieces * a.piece < V || a.piece >= 1 << 23) bad = 14;
        if (bad) { printf("%d: rows %lld d %d V %d n %d\n", bad, (long long)rows, d, V, n); return 1; }
    }
    puts("fits");
}
""")
    hipcc = os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "bin", "hipcc")
    lib = os.path.dirname(capi.LIB)
    subprocess.run([hipcc, "-x", "hip", "--offload-host-only", "-O2", "-std=c++17", str(src), "-o", str(tmp_path / "plans"),
                    f"-L{lib}", "-lfa2_mi355x", f"-Wl,-rpath,{lib}"], check=True, capture_output=True)
    out = subprocess.run([str(tmp_path / "plans")], capture_output=True, text=True)
    assert out.returncode == 0 and "fits" in out.stdout, out.stdout
