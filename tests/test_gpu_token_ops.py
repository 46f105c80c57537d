"""The operators on token rows as they are used together: a decoder's training step and its cached serving path through
them against the same weights on torch's operators; streams, captured graphs, two calls in flight."""
import pytest
import torch

import fa2_decoder as dec

pytestmark = pytest.mark.gpu
DEV = "cuda"


def rel(a, b):
    return ((a.double() - b.double()).norm() / b.double().norm()).item()


def models(fa, vocab=1000, n_layers=2, d_ff=512, **kw):
    torch.manual_seed(0)
    a = dec.Decoder(vocab=vocab, n_layers=n_layers, d_ff=d_ff, fa=fa, fused=True, **kw).to(DEV)
    b = dec.Decoder(vocab=vocab, n_layers=n_layers, d_ff=d_ff, fa=fa).to(DEV)
    b.load_state_dict(a.state_dict())
    return a, b


@pytest.mark.parametrize("B,S,vocab", [(2, 320, 1000), (1, 33, 1003), (4, 700, 5000)])
def test_training_step(fa, B, S, vocab):
    """fp16 autocast with a scaled loss: the same loss and gradients as the unfused model.  Both round every branch and
    norm to fp16 (2^-11 each, about ten of them in a row per block): 1e-2 as for the attention's drop-in test."""
    a, b = models(fa, vocab)
    ids = dec.synthetic_ids(B, S, vocab=vocab, seed=1, device=DEV)
    losses = []
    for m in (a, b):
        with torch.autocast("cuda", dtype=torch.float16):
            loss = m.loss(ids)
        (loss * 1024).backward()
        losses.append(loss.item())
    assert abs(losses[0] - losses[1]) < 1e-3 * abs(losses[1])
    for (n, pa), (_, pb) in zip(a.named_parameters(), b.named_parameters()):
        assert pa.grad.dtype == torch.float32 and rel(pa.grad, pb.grad) < 1e-2, n


def test_training_step_with_dropout(fa):
    """Dropout runs in training only, with a new mask each step, and leaves finite gradients everywhere."""
    a, b = models(fa, dropout=0.1)
    ids = dec.synthetic_ids(2, 200, vocab=1000, seed=1, device=DEV)
    with torch.autocast("cuda", dtype=torch.float16):
        first, second = a.loss(ids), a.loss(ids)
        second.backward()
        a.eval()
        plain, ref = a.loss(ids), b.loss(ids)
    assert first.item() != second.item() and abs(plain.item() - ref.item()) < 1e-3 * ref.item()
    assert all(torch.isfinite(p.grad).all() and p.grad.abs().max() > 0 for p in a.parameters())


def test_cached_serving(fa):
    """A prefill chunk and single tokens against the unfused model's logits; then with 8-bit projections, whose weights and
    rows are each off by up to 2^-4 of a value at random (about 2^-5.8 in the mean square each, so 2.6% a product)."""
    a, b = models(fa)
    a, b = a.half().eval(), b.half().eval()
    ids = dec.synthetic_ids(3, 47, vocab=1000, seed=2, device=DEV)
    with torch.no_grad():
        def logits(m):
            cache = m.new_cache()
            out = [m.forward_cached(ids[:, :40], cache, 64)]
            out += [m.forward_cached(ids[:, i:i + 1], cache, 64) for i in range(40, 48)]
            return torch.cat(out, 1)
        ra, rb = logits(a), logits(b)
        assert ra.shape == (3, 48, 1000) and rel(ra, rb) < 5e-3
        r8 = logits(a.quantize())
    assert torch.isfinite(r8).all() and 1e-3 < rel(r8, rb) < 0.1


def calls(fa, seed, dtype=torch.float16, n=300, d=128, V=700):
    """A set of inputs and the run of all operators on them, forward and backward, as a step makes it."""
    g = torch.Generator().manual_seed(seed)
    x, r = (torch.randn(n, d, generator=g).to(t).to(DEV).requires_grad_(True) for t in (dtype, torch.float32))
    w = torch.rand(d, generator=g).to(DEV).requires_grad_(True)
    head = (torch.randn(V, d, generator=g) * 0.1).to(dtype).to(DEV).requires_grad_(True)
    target = torch.randint(0, V, (n,), generator=g)
    target[::7] = -100
    target = target.to(DEV)
    scale = torch.tensor(256.0, device=DEV)

    def run():
        y, h = fa.add_rms_norm(x, r, w, dropout_p=0.1, seed=seed)
        z = fa.dropout(fa.rms_norm(h, w, out_dtype=dtype), 0.2, seed=seed + 1)
        loss = fa.linear_cross_entropy(y + z, head, target)
        grads = torch.autograd.grad(loss, (x, r, w, head), scale)
        with torch.no_grad():
            q, s, h2 = fa.rms_norm_fp8(x.detach(), w.detach(), residual=r.detach())
        return [loss.detach(), *grads, q.float(), s, h2]

    return run, (x, r, w, head, target)


def test_other_streams_and_two_calls_in_flight(fa):
    runs = [calls(fa, s)[0] for s in range(4)]
    ref = [r() for r in runs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    got = []
    for r, s in zip(runs, streams):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(r())
    torch.cuda.synchronize()
    for a, b in zip(got, ref):
        assert all(torch.equal(u, v) for u, v in zip(a, b))


def test_captured_graphs(fa):
    """Two graphs of different inputs, replayed in turn with eager work and new inputs between the replays."""
    captured = []
    for seed in range(2):
        run, inputs = calls(fa, seed)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            run()
        torch.cuda.current_stream().wait_stream(s)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = run()
        captured.append((g, out, run, inputs))
    for it in range(3):
        for g, out, run, inputs in captured:
            with torch.no_grad():
                for t in inputs[:4]:
                    t.copy_(torch.randn(t.shape, device=DEV) * (0.1 if t is inputs[3] else 1.0))
                inputs[4].copy_(torch.where(torch.rand(inputs[4].shape, device=DEV) < 0.3, -100, inputs[4].clamp_min(0) + it))
            g.replay()
            torch.cuda.synchronize()
            first = [t.clone() for t in out]
            eager = run()
            g.replay()
            torch.cuda.synchronize()
            for a, b, c in zip(first, eager, out):
                assert torch.equal(a, b) and torch.equal(c, b)


def test_saved_tensors_are_watched(fa):
    """Changing what the backward needs, in place, is an error and not a wrong gradient."""
    x = torch.randn(20, 64, device=DEV).half().requires_grad_(True)
    w = torch.ones(64, device=DEV)
    head = torch.randn(50, 64, device=DEV).half()
    y, h = fa.add_rms_norm(x, torch.zeros_like(x), w)
    h.add_(1)
    with pytest.raises(RuntimeError):
        y.sum().backward()
    loss = fa.linear_cross_entropy(x, head, torch.zeros(20, dtype=torch.long, device=DEV))
    head.mul_(2)
    with pytest.raises(RuntimeError):
        loss.backward()


def test_refused_second_derivative(fa):
    x = torch.randn(20, 64, device=DEV).half().requires_grad_(True)
    head = torch.randn(50, 64, device=DEV).half()
    for y in (fa.linear_cross_entropy(x, head, torch.zeros(20, dtype=torch.long, device=DEV)), fa.dropout(x, 0.1).float().sum()):
        (g,) = torch.autograd.grad(y, x, create_graph=True)
        with pytest.raises(RuntimeError):
            g.float().sum().backward()
