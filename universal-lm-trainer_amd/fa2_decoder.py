"""Minimal pre-norm decoder in the reference's shape, used to exercise the
attention path inside a full training step (benchmark configuration 5) and in
the model-level drop-in test; with ``fused=True`` it also runs what lies between
two attention calls, and the loss, through the package's operators on token rows.

It mirrors what reaches the attention kernel in the reference
(reference @ None: train.py:1861-2105) -- fused QKV projection, q/k/v as
(B,S,H,D) views transposed to (B,H,S,D), fused RoPE through
``flash_attn_v100_cuda.rope`` (eager fallback otherwise), attention through
``flash_attn_v100_cuda.flash_attn_v100`` (SDPA fallback otherwise),
``attn.transpose(1,2).contiguous().view(B,S,D)`` and the output projection --
plus RMSNorm, a SwiGLU FFN and a tied LM head.  It is a consumer of the path,
not a reimplementation of the reference's training runtime.
"""

import torch
import torch.nn as nn
import torch.nn.functional as F

import fa2_workloads as wl


def rotate_half(x):
    x1, x2 = x.chunk(2, dim=-1)
    return torch.cat((-x2, x1), dim=-1)


class Attention(nn.Module):
    def __init__(self, d_model, n_heads, fa=None, use_kernel=True):
        super().__init__()
        self.h, self.d = n_heads, d_model // n_heads
        self.wqkv = nn.Linear(d_model, 3 * d_model, bias=False)
        self.wo = nn.Linear(d_model, d_model, bias=False)
        self.fa, self.use_kernel = fa, use_kernel
        self.attn_fn = None  # optional override (q, k, v) -> o, used for timing
        # Fallback path only: attention through SDPA's math backend in fp32 (the
        # reference path the kernel's parity is defined against), cast back.
        self.ref_fp32 = False

    def forward(self, x, cos, sin):
        B, S, D = x.shape
        q, k, v = self.wqkv(x).chunk(3, dim=-1)
        q = q.view(B, S, self.h, self.d).transpose(1, 2)
        k = k.view(B, S, self.h, self.d).transpose(1, 2)
        v = v.view(B, S, self.h, self.d).transpose(1, 2)
        fa = self.fa if self.use_kernel else None
        if fa is not None and fa.rope_can_use(q, k, cos, sin):
            q, k = fa.rope(q, k, cos, sin)
        else:
            c, s = cos[None, None], sin[None, None]
            q, k = q * c + rotate_half(q) * s, k * c + rotate_half(k) * s
        if torch.is_autocast_enabled():
            q, k, v = (t.half() if t.dtype == torch.float32 else t for t in (q, k, v))
        if fa is not None and fa.can_use(q, k, v):
            attn = self.attn_fn(q, k, v) if self.attn_fn else fa.flash_attn_v100(q, k, v, causal=True)
        elif self.ref_fp32:
            from torch.nn.attention import SDPBackend, sdpa_kernel
            with torch.autocast(x.device.type, enabled=False), sdpa_kernel(SDPBackend.MATH):
                attn = F.scaled_dot_product_attention(q.float(), k.float(), v.float(), is_causal=True).to(q.dtype)
        else:
            attn = F.scaled_dot_product_attention(q, k, v, is_causal=True)
        return self.wo(attn.transpose(1, 2).contiguous().view(B, S, D))

    def forward_cached(self, x, cos, sin, cache):
        """Inference: x holds the last S_new positions of the sequence, cos/sin
        their RoPE rows, and cache = [k, v] the earlier positions' rotated keys
        and values ((B,H,S_past,64) each, or None), extended in place.  The
        queries see every cached key and the causal part of their own: the
        bottom-right mask an HF-style KV-cache decoder builds
        (reference @ None: hf_template/modeling_universal_lm.py:228-251),
        through ``flash_attn_kvcache`` or, on the fallback path, SDPA with
        that mask spelled out."""
        return self.cached(self.wqkv(x), cos, sin, cache)

    def cached(self, qkv, cos, sin, cache):
        """forward_cached from the fused QKV projection's output on."""
        B, S, D = *qkv.shape[:2], qkv.shape[2] // 3
        q, k, v = (t.view(B, S, self.h, self.d).transpose(1, 2) for t in qkv.chunk(3, dim=-1))
        fa = self.fa if self.use_kernel else None
        if fa is not None and fa.rope_can_use(q, k, cos, sin):
            q, k = fa.rope(q, k, cos, sin)
        else:
            c, s = cos[None, None], sin[None, None]
            q, k = ((t * c + rotate_half(t) * s).to(v.dtype) for t in (q, k))
        if cache[0] is not None:
            k, v = torch.cat([cache[0], k], dim=2), torch.cat([cache[1], v], dim=2)
        cache[0], cache[1] = k, v
        if fa is not None:
            attn = fa.flash_attn_kvcache(q, k, v, causal=True)
        else:
            Sk = k.shape[2]
            mask = torch.ones(S, Sk, dtype=torch.bool, device=qkv.device).tril(Sk - S)
            attn = F.scaled_dot_product_attention(q, k, v, attn_mask=mask)
        return self.wo(attn.transpose(1, 2).contiguous().view(B, S, D))


class Proj8:
    """A linear layer's weight in e4m3 with one scale an output, for rows that
    ``rms_norm_fp8`` left in 8 bits; the product is the library's."""

    def __init__(self, linear):
        w = linear.weight.detach().float()
        scale = (w.abs().amax(1, keepdim=True) / 448).clamp_min(2.0 ** -126)
        self.w, self.scale = (w / scale).to(torch.float8_e4m3fn), scale.t().contiguous()

    def __call__(self, q, scale, dtype):
        y = torch._scaled_mm(q.reshape(-1, q.shape[-1]), self.w.t(), scale_a=scale.reshape(-1, 1), scale_b=self.scale,
                             out_dtype=torch.bfloat16)   # the only output type of row-wise scales
        return y.view(*q.shape[:-1], -1).to(dtype)


class Block(nn.Module):
    def __init__(self, d_model, n_heads, d_ff, fa, use_kernel):
        super().__init__()
        self.fa = fa
        self.proj8 = None   # (wqkv, w1, w3) in 8 bits, for forward_cached_fused
        self.n1 = nn.RMSNorm(d_model, eps=1e-6)
        self.n2 = nn.RMSNorm(d_model, eps=1e-6)
        self.attn = Attention(d_model, n_heads, fa, use_kernel)
        self.w1 = nn.Linear(d_model, d_ff, bias=False)
        self.w3 = nn.Linear(d_model, d_ff, bias=False)
        self.w2 = nn.Linear(d_ff, d_model, bias=False)

    def forward(self, x, cos, sin):
        x = x + self.attn(self.n1(x), cos, sin)
        h = self.n2(x)
        return x + self.w2(F.silu(self.w1(h)) * self.w3(h))

    def forward_cached(self, x, cos, sin, cache):
        x = x + self.attn.forward_cached(self.n1(x), cos, sin, cache)
        h = self.n2(x)
        return x + self.w2(F.silu(self.w1(h)) * self.w3(h))

    def norm(self, n, branch, h, p):
        """The last branch (None before the first block) added to the residual stream h
        and the norm n of the sum: (y, h), y of the type the next linear layer takes."""
        if branch is None:
            dtype = torch.get_autocast_dtype("cuda") if torch.is_autocast_enabled("cuda") else h.dtype
            return self.fa.rms_norm(h, n.weight, eps=n.eps, out_dtype=dtype), h
        return self.fa.add_rms_norm(branch, h, n.weight, eps=n.eps, dropout_p=p)

    def forward_fused(self, branch, h, cos, sin, p):
        """forward with the residual stream h and the branch that is still to be added
        kept apart; returns the pair."""
        y, h = self.norm(self.n1, branch, h, p)
        y, h = self.norm(self.n2, self.attn(y, cos, sin), h, p)
        return self.w2(F.silu(self.w1(y)) * self.w3(y)), h

    def norm8(self, n, branch, h):
        """norm in 8 bits, without dropout: (q, scale, h)."""
        if branch is None:
            return (*self.fa.rms_norm_fp8(h, n.weight, eps=n.eps), h)
        return self.fa.rms_norm_fp8(branch, n.weight, eps=n.eps, residual=h)

    def forward_cached_fused(self, branch, h, cos, sin, cache):
        if self.proj8 is None:
            y, h = self.norm(self.n1, branch, h, 0.0)
            y, h = self.norm(self.n2, self.attn.forward_cached(y, cos, sin, cache), h, 0.0)
            return self.w2(F.silu(self.w1(y)) * self.w3(y)), h
        wqkv, w1, w3 = self.proj8
        q, s, h = self.norm8(self.n1, branch, h)
        a = self.attn.cached(wqkv(q, s, h.dtype), cos, sin, cache)
        q, s, h = self.norm8(self.n2, a, h)
        return self.w2(F.silu(w1(q, s, h.dtype)) * w3(q, s, h.dtype)), h


class Decoder(nn.Module):
    """``fused``: norms, residual additions, dropout and the loss through the package's
    operators (GPU; the residual stream and its next branch are kept apart between
    blocks).  ``dropout`` (with ``fused``): of the embedding and of every branch, in
    training."""

    def __init__(self, vocab=32000, d_model=768, n_heads=12, n_layers=10, d_ff=2048, fa=None, use_kernel=True,
                 fused=False, dropout=0.0):
        super().__init__()
        if fused and fa is None or dropout and not fused:
            raise ValueError("fused needs the kernel module, and dropout needs fused")
        self.fa, self.fused, self.dropout = fa, fused, dropout
        self.emb = nn.Embedding(vocab, d_model)
        self.layers = nn.ModuleList(Block(d_model, n_heads, d_ff, fa, use_kernel) for _ in range(n_layers))
        self.norm = nn.RMSNorm(d_model, eps=1e-6)
        self.head_dim = d_model // n_heads
        self.d_model = d_model
        for p in self.parameters():  # std 0.02 init (train.py:2015-2022)
            nn.init.normal_(p, std=0.02) if p.dim() > 1 else nn.init.ones_(p)

    def forward_hidden(self, ids):
        """The final norm's output, which the tied head takes."""
        S = ids.shape[1]
        cos, sin = wl.rope_tables(S, d_model=self.d_model, head_dim=self.head_dim)
        cos, sin = cos.to(ids.device), sin.to(ids.device)
        x = self.emb(ids)
        if self.fused:
            p = self.dropout if self.training else 0.0
            branch, h = None, self.fa.dropout(x, p)
            for layer in self.layers:
                branch, h = layer.forward_fused(branch, h, cos, sin, p)
            return self.layers[-1].norm(self.norm, branch, h, p)[0]
        for layer in self.layers:
            x = layer(x, cos, sin)
        return self.norm(x)

    def forward(self, ids):
        return F.linear(self.forward_hidden(ids), self.emb.weight)  # tied head

    def quantize(self):
        """Projections behind a norm in 8 bits from now on, in cached (serving) calls of a
        fused model: a copy of the weights as they are, on their device."""
        if not self.fused:
            raise ValueError("8-bit projections need fused")
        for layer in self.layers:
            layer.proj8 = tuple(Proj8(m) for m in (layer.attn.wqkv, layer.w1, layer.w3))
        return self

    def new_cache(self):
        return [[None, None] for _ in self.layers]

    def forward_cached(self, ids, cache, max_len):
        """Logits of the S_new tokens ``ids`` that follow the positions held in
        ``cache`` (from ``new_cache()``, extended in place): a prefill chunk or
        one decode step.  ``max_len`` sizes the RoPE tables."""
        past = 0 if cache[0][0] is None else cache[0][0].shape[2]
        S = ids.shape[1]
        cos, sin = wl.rope_tables(max_len, d_model=self.d_model, head_dim=self.head_dim)
        cos, sin = (t[past:past + S].contiguous().to(ids.device) for t in (cos, sin))
        x = self.emb(ids)
        if self.fused:
            branch, h = None, x
            for layer, c in zip(self.layers, cache):
                branch, h = layer.forward_cached_fused(branch, h, cos, sin, c)
            return F.linear(self.layers[-1].norm(self.norm, branch, h, 0.0)[0], self.emb.weight)
        for layer, c in zip(self.layers, cache):
            x = layer.forward_cached(x, cos, sin, c)
        return F.linear(self.norm(x), self.emb.weight)

    def loss(self, ids):
        if self.fused:
            return self.fa.linear_cross_entropy(self.forward_hidden(ids[:, :-1]), self.emb.weight, ids[:, 1:])
        logits = self.forward(ids[:, :-1])
        return F.cross_entropy(logits.float().reshape(-1, logits.shape[-1]), ids[:, 1:].reshape(-1))


def compare_training_step(fa, B, S, n_layers=10, d_ff=2048, vocab=32000, seed=0, device="cuda"):
    """One fp16-autocast training step (GradScaler-scaled backward, then unscaled
    gradients) of the same random-init weights through the kernel path
    (``flash_attn_v100`` + fused ``rope``) and through the reference path (eager
    RoPE, attention by SDPA's math backend in fp32), as train.py's loop runs it
    (reference @ None: train.py:1931-1964, 2341-2424).  Returns (loss_kernel,
    loss_reference, {parameter name: relative L2 error of its gradient})."""
    torch.manual_seed(seed)
    mk = Decoder(vocab=vocab, n_layers=n_layers, d_ff=d_ff, fa=fa, use_kernel=True).to(device)
    mr = Decoder(vocab=vocab, n_layers=n_layers, d_ff=d_ff, fa=None, use_kernel=False).to(device)
    mr.load_state_dict(mk.state_dict())
    for layer in mr.layers:
        layer.attn.ref_fp32 = True
    ids = synthetic_ids(B, S, vocab=vocab, seed=seed + 1, device=device)
    losses = []
    for m in (mk, mr):
        opt = torch.optim.SGD(m.parameters(), lr=0.0)
        scaler = torch.amp.GradScaler(device, init_scale=2.0 ** 16)
        with torch.autocast(device, dtype=torch.float16):
            loss = m.loss(ids)
        scaler.scale(loss).backward()
        scaler.unscale_(opt)
        losses.append(loss.item())
    errs = {}
    for (n, pk), (_, pr) in zip(mk.named_parameters(), mr.named_parameters()):
        errs[n] = ((pk.grad.float() - pr.grad.float()).norm() / pr.grad.float().norm()).item()
    del mk, mr
    return losses[0], losses[1], errs


def synthetic_ids(B, S, vocab=32000, seed=0, device="cpu"):
    g = torch.Generator("cpu").manual_seed(seed)
    return torch.randint(0, vocab, (B, S + 1), generator=g).to(device)


def step_flops_attention(B, S, H=12, D=64, n_layers=10):
    f, b = wl.causal_flops(B, H, S, D)
    return n_layers * (f + b)


def approx_step_flops(B, S, d_model=768, d_ff=2048, n_layers=10, vocab=32000):
    """6 * params_active * tokens for the linear layers and head, plus attention."""
    lin = n_layers * (4 * d_model * d_model + 3 * d_model * d_ff) + vocab * d_model
    return 6 * lin * B * S + step_flops_attention(B, S, d_model // 64, 64, n_layers)

