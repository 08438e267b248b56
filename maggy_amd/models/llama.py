"""Llama-3-style decoder-only transformer (RMSNorm / SwiGLU / RoPE / GQA).

Llama-3 8B bf16 data-parallel over 8x MI355X.
Self-contained (no transformers dependency); random-init weights, synthetic
token data.  Attention goes through torch.nn.functional
scaled_dot_product_attention, which on ROCm dispatches to the fused
(AOTriton/composable-kernel) kernels when available and the math path
otherwise.  The 288 GB HBM3E per GPU fits the full 8B model + Adam states
without sharding, so plain DP is the natural parallelism.
"""
import functools
import math
import threading
from dataclasses import dataclass

import torch
import torch.nn as nn
import torch.nn.functional as F

from maggy_amd.ops.block8 import (
    Linear8Group,
    Linear8Member,
    MaggyFeedForward8,
    MaggyRMSNorm8,
    groups8,
)
from maggy_amd.ops.fused_rms import (  # noqa: F401
    MaggyRMSNorm,
    rope_bthd,
    swiglu,
)
from maggy_amd.ops.linear import MaggyFeedForward, MaggyLinear


@dataclass
class LlamaConfig:
    vocab_size: int = 128256
    dim: int = 4096
    n_layers: int = 32
    n_heads: int = 32
    n_kv_heads: int = 8
    ffn_hidden: int = 14336
    max_seq_len: int = 8192
    rope_theta: float = 500000.0
    norm_eps: float = 1e-5
    # the layers' projections, feed-forwards and norms on the 8-bit block
    # operators (ops/block8.py); embeddings, attention and lm_head stay
    eight_bit: bool = False

    @staticmethod
    def llama3_8b():
        return LlamaConfig()

    @staticmethod
    def tiny(vocab_size=512):
        """CPU-testable toy config."""
        return LlamaConfig(vocab_size=vocab_size, dim=64, n_layers=2,
                           n_heads=4, n_kv_heads=2, ffn_hidden=128,
                           max_seq_len=128)

    @staticmethod
    def small_1b():
        """Llama-3.2-1B-ish shape for single-GPU experiments."""
        return LlamaConfig(vocab_size=128256, dim=2048, n_layers=16,
                           n_heads=32, n_kv_heads=8, ffn_hidden=8192)


# RMSNorm: the fused HIP kernel on GPU bf16, eager fp32 math elsewhere
RMSNorm = MaggyRMSNorm


def precompute_rope(dim, max_seq_len, theta):
    inv_freq = 1.0 / (theta ** (torch.arange(0, dim, 2).float() / dim))
    t = torch.arange(max_seq_len).float()
    freqs = torch.outer(t, inv_freq)
    return torch.cos(freqs), torch.sin(freqs)


def apply_rope(x, cos, sin, pos=0):
    # x: [B, H, T, D]; rotate pairs (x0,x1) in the last dim; ``pos`` is
    # the absolute position of x's first token (KV-cached decode)
    T = x.shape[-2]
    cos = cos[pos:pos + T].to(x.dtype)
    sin = sin[pos:pos + T].to(x.dtype)
    x1, x2 = x[..., 0::2], x[..., 1::2]
    out = torch.empty_like(x)
    out[..., 0::2] = x1 * cos - x2 * sin
    out[..., 1::2] = x2 * cos + x1 * sin
    return out


def _sdpa(q, k, v, causal, gqa):
    """SDPA with a measured ROCm backend choice (override with
    MAGGY_SDPA=flash|efficient|math).

    The attention BACKWARD was 20% of the 8B training step with the
    default flash (AOTriton) dispatch — bwd_kernel_dk_dv+dq ran at ~57%
    of the forward's efficiency (profiles/r10).  The CK memory-efficient
    backend's backward is ~2x faster: 18,626 vs 16,346 tokens/sec
    end-to-end (+14%), measured at b4 x 4096 on one MI355X — so TRAINING
    (grad-enabled) prefill uses `efficient` by default, including the
    KV-head expansion it needs for GQA.  Inference/decode keeps the
    flash forward (fastest fwd-only)."""
    import os

    choice = os.environ.get("MAGGY_SDPA", "")
    if not choice and q.is_cuda and q.requires_grad and causal:
        choice = "efficient"
    if choice:
        from torch.nn.attention import SDPBackend, sdpa_kernel

        backend = {"flash": SDPBackend.FLASH_ATTENTION,
                   "efficient": SDPBackend.EFFICIENT_ATTENTION,
                   "math": SDPBackend.MATH}[choice]
        if choice == "efficient" and gqa:
            # CK mem-efficient path has no enable_gqa: expand KV heads
            rep = q.shape[1] // k.shape[1]
            k = k.repeat_interleave(rep, dim=1)
            v = v.repeat_interleave(rep, dim=1)
            gqa = False
        with sdpa_kernel([backend, SDPBackend.MATH]):
            return F.scaled_dot_product_attention(
                q, k, v, is_causal=causal, enable_gqa=gqa)
    return F.scaled_dot_product_attention(
        q, k, v, is_causal=causal, enable_gqa=gqa)


class Attention(nn.Module):
    def __init__(self, cfg):
        super().__init__()
        self.n_heads = cfg.n_heads
        self.n_kv_heads = cfg.n_kv_heads
        self.head_dim = cfg.dim // cfg.n_heads
        # MaggyLinear = nn.Linear running on the in-tree MFMA GEMM
        # (fwd + both backward layouts) when the shapes tile; eager/rocBLAS
        # fallback otherwise (tiny CPU configs)
        linear = Linear8Member if cfg.eight_bit else MaggyLinear
        self.wq = linear(cfg.dim, cfg.n_heads * self.head_dim)
        self.wk = linear(cfg.dim, cfg.n_kv_heads * self.head_dim)
        self.wv = linear(cfg.dim, cfg.n_kv_heads * self.head_dim)
        self.wo = linear(cfg.n_heads * self.head_dim, cfg.dim)
        self.qkv8 = self.out8 = None
        if cfg.eight_bit:
            self.qkv8 = Linear8Group(self, "wq", "wk", "wv")
            self.out8 = Linear8Group(self, "wo")

    def _project_out(self, x):
        return self.wo(x) if self.out8 is None else self.out8(x)

    def forward(self, x, cos, sin, cache=None, pos=0):
        B, T, _ = x.shape
        # RoPE applies on the [B, T, H, D] layout BEFORE the head
        # transpose (one fused bf16 pass, ops/fused_rms.py::rope_bthd)
        if self.qkv8 is None:
            q, k, v = self.wq(x), self.wk(x), self.wv(x)
        else:
            q, k, v = self.qkv8(x)
        q = q.view(B, T, self.n_heads, self.head_dim)
        k = k.view(B, T, self.n_kv_heads, self.head_dim)
        v = v.view(B, T, self.n_kv_heads, self.head_dim).transpose(1, 2)
        q = rope_bthd(q, cos, sin, pos).transpose(1, 2)
        k = rope_bthd(k, cos, sin, pos).transpose(1, 2)
        if cache is not None:
            # STATIC KV cache (decode path): preallocated [B, KV, cap, D]
            # buffers written in place — the torch.cat idiom re-copies the
            # whole cache every decoded token (~1 GB/token at 8B b8)
            if cache.get("kbuf") is None:
                cap = int(cache.get("cap", pos + T + 256))
                # zeros: the masked step reads all of it, and a masked value
                # times a NaN that happens to be there is NaN
                cache["kbuf"] = k.new_zeros(
                    B, self.n_kv_heads, cap, self.head_dim)
                cache["vbuf"] = v.new_zeros(
                    B, self.n_kv_heads, cap, self.head_dim)
                cache["len"] = 0
            if cache.get("idx") is not None:
                # hipGraph-capturable step (T == 1): the write position
                # and attention mask live in DEVICE buffers updated
                # between replays, so no python int is baked into the
                # capture; attention runs masked over the full capacity
                return self._masked_decode_step(x.shape[0], q, k, v, cache)
            L = cache["len"]
            cache["kbuf"][:, :, L:L + T] = k
            cache["vbuf"][:, :, L:L + T] = v
            cache["len"] = L + T
            k = cache["kbuf"][:, :, :L + T]
            v = cache["vbuf"][:, :, :L + T]
        # causal masking is needed only when the query block spans >1 new
        # position; a single decoded token attends to the whole cache
        causal = T > 1
        out = _sdpa(q, k, v, causal, self.n_kv_heads != self.n_heads)
        out = out.transpose(1, 2).reshape(B, T, -1)
        return self._project_out(out)

    def _masked_decode_step(self, B, q, k, v, cache):
        """Capture-safe single-token attention: in-place index_copy of
        the new KV at the device-resident position, bmm attention over
        the FULL cache capacity with an additive -inf mask (the few
        masked tail columns cost ~nothing; every op here is hipGraph
        recordable)."""
        idx, mask = cache["idx"], cache["mask"]
        kbuf, vbuf = cache["kbuf"], cache["vbuf"]
        kbuf.index_copy_(2, idx, k)
        vbuf.index_copy_(2, idx, v)
        rep = self.n_heads // self.n_kv_heads
        scale = 1.0 / math.sqrt(self.head_dim)
        # q: [B, H, 1, D] -> [B, KV, rep, D]
        q4 = q.reshape(B, self.n_kv_heads, rep, self.head_dim)
        scores = torch.einsum("bkrd,bksd->bkrs", q4, kbuf) * scale
        scores = scores + mask  # [1,1,1,cap] broadcast; -inf beyond len
        probs = scores.float().softmax(-1).to(q.dtype)
        outh = torch.einsum("bkrs,bksd->bkrd", probs, vbuf)
        out = outh.reshape(B, 1, self.n_heads * self.head_dim)
        return self._project_out(out)


class FeedForward(MaggyFeedForward):
    """Llama MLP: custom-GEMM w1/w3 with the SwiGLU fused into the w3
    GEMM's epilogue (ops/linear.py); eager fallback off-GPU."""

    def __init__(self, cfg):
        super().__init__(cfg.dim, cfg.ffn_hidden)


class Block(nn.Module):
    def __init__(self, cfg):
        super().__init__()
        norm = MaggyRMSNorm8 if cfg.eight_bit else RMSNorm
        self.attn_norm = norm(cfg.dim, cfg.norm_eps)
        self.attn = Attention(cfg)
        self.ffn_norm = norm(cfg.dim, cfg.norm_eps)
        self.ffn = MaggyFeedForward8(cfg.dim, cfg.ffn_hidden) \
            if cfg.eight_bit else FeedForward(cfg)

    def forward(self, x, cos, sin, cache=None, pos=0):
        x = x + self.attn(self.attn_norm(x), cos, sin, cache=cache, pos=pos)
        x = x + self.ffn(self.ffn_norm(x))
        return x


def _packed_while(generate):
    """Decode with the 8-bit weights packed once a call, for this thread
    alone, unless what the caller has packed (``pack8_model``) still holds
    for them."""
    @functools.wraps(generate)
    def run(self, *args, **kw):
        me, made, kept = threading.get_ident(), [], []
        try:
            for g in groups8(self):
                packed, fresh = g.pack_own()
                if fresh:
                    made.append(g)
                # a graph that generate captures reads these to its end
                kept.append(packed)
            return generate(self, *args, **kw)
        finally:
            for g in made:
                g.drop_own(me)
    return run


class LlamaModel(nn.Module):
    def __init__(self, cfg):
        super().__init__()
        self.cfg = cfg
        self.tok_emb = nn.Embedding(cfg.vocab_size, cfg.dim)
        self.layers = nn.ModuleList(Block(cfg) for _ in range(cfg.n_layers))
        self.norm = RMSNorm(cfg.dim, cfg.norm_eps)
        self.lm_head = MaggyLinear(cfg.dim, cfg.vocab_size)
        cos, sin = precompute_rope(cfg.dim // cfg.n_heads, cfg.max_seq_len,
                                   cfg.rope_theta)
        self.register_buffer("rope_cos", cos, persistent=False)
        self.register_buffer("rope_sin", sin, persistent=False)
        self.apply(self._init)

    def _init(self, m):
        if isinstance(m, nn.Linear):
            nn.init.normal_(m.weight, std=0.02 / math.sqrt(
                2 * self.cfg.n_layers))
        elif isinstance(m, nn.Embedding):
            nn.init.normal_(m.weight, std=0.02)

    def forward(self, tokens, targets=None):
        x = self.tok_emb(tokens)
        for layer in self.layers:
            x = layer(x, self.rope_cos, self.rope_sin)
        x = self.norm(x)
        if targets is not None:
            logits = self.lm_head(x)
            # bf16 logits straight into CE: torch accumulates the softmax
            # reduction in fp32, and skipping the fp32 materialization of
            # the [tokens, vocab] logits saves ~3.4x on the loss kernels
            return F.cross_entropy(
                logits.view(-1, logits.size(-1)), targets.view(-1)
            ).float()
        return self.lm_head(x)

    def num_params(self):
        return sum(p.numel() for p in self.parameters())

    @torch.no_grad()
    @_packed_while
    def generate(self, tokens, max_new_tokens, temperature=0.0, top_k=None):
        """KV-cached autoregressive decoding (greedy at temperature 0).

        :param tokens: [B, T_prompt] prompt ids
        :returns: [B, T_prompt + max_new_tokens] ids
        """
        self.eval()
        cap = tokens.shape[1] + max_new_tokens
        caches = [{"kbuf": None, "cap": cap} for _ in self.layers]
        out = tokens
        x_in = tokens
        pos = 0
        for _ in range(max_new_tokens):
            x = self.tok_emb(x_in)
            for layer, cache in zip(self.layers, caches):
                x = layer(x, self.rope_cos, self.rope_sin, cache=cache,
                          pos=pos)
            logits = self.lm_head(self.norm(x[:, -1:, :]))[:, -1, :]
            if temperature > 0:
                logits = logits / temperature
                if top_k is not None:
                    kth = torch.topk(logits, top_k, dim=-1).values[..., -1:]
                    logits = logits.masked_fill(logits < kth,
                                                float("-inf"))
                probs = torch.softmax(logits.float(), dim=-1)
                nxt = torch.multinomial(probs, 1)
            else:
                nxt = logits.argmax(dim=-1, keepdim=True)
            pos += x_in.shape[1]
            out = torch.cat([out, nxt], dim=1)
            x_in = nxt
        return out

    @torch.no_grad()
    @_packed_while
    def generate_captured(self, tokens, max_new_tokens, use_graph=True):
        """Greedy decode with a hipGraph-captured per-token step
        (EXPERIMENTAL: measured 868 vs 929 tok/s against the eager
        static-cache path at 8B — the masked full-capacity attention
        costs more than the launch gaps it saves — and graph capture is
        sensitive to process-wide CUDA state; ``generate`` remains the
        production decode path).

        The decode step's inputs live in STATIC device buffers (input
        token, KV write index, attention mask, per-position RoPE row);
        the loop updates those buffers and replays one graph per token —
        ~400 kernel launches collapse into one replay at 8B.  With
        ``use_graph=False`` the same static-buffer masked path runs
        eagerly (CPU-testable; numerically identical).
        """
        self.eval()
        B, Tp = tokens.shape
        cap = Tp + max_new_tokens
        caches = [{"kbuf": None, "cap": cap} for _ in self.layers]
        # eager prefill fills cache[0:Tp]
        x = self.tok_emb(tokens)
        for layer, c in zip(self.layers, caches):
            x = layer(x, self.rope_cos, self.rope_sin, cache=c, pos=0)
        logits = self.lm_head(self.norm(x[:, -1:, :]))[:, -1, :]
        cur = logits.argmax(dim=-1, keepdim=True)
        outs = [tokens, cur]
        if max_new_tokens == 1:
            return torch.cat(outs, dim=1)

        dev = tokens.device
        x_in = cur.clone()
        idx = torch.full((1,), Tp, device=dev, dtype=torch.long)
        mask = torch.full((1, 1, 1, cap), float("-inf"), device=dev,
                          dtype=torch.float32)
        mask[..., :Tp + 1] = 0.0
        cos_step = self.rope_cos[Tp:Tp + 1].clone()
        sin_step = self.rope_sin[Tp:Tp + 1].clone()
        for c in caches:
            c["idx"] = idx
            c["mask"] = mask

        def step():
            h = self.tok_emb(x_in)
            for layer, c in zip(self.layers, caches):
                h = layer(h, cos_step, sin_step, cache=c, pos=0)
            lg = self.lm_head(self.norm(h))[:, -1, :]
            return lg.argmax(dim=-1, keepdim=True)

        if use_graph and tokens.is_cuda:
            s = torch.cuda.Stream()
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                step()  # warmup (positions re-written by the real loop)
            torch.cuda.current_stream().wait_stream(s)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                nxt_static = step()

            def run_step():
                graph.replay()
                return nxt_static
        else:
            run_step = step

        for i in range(max_new_tokens - 1):
            p = Tp + i  # position of the token in x_in
            x_in.copy_(cur)
            idx.fill_(p)
            mask[..., p] = 0.0
            cos_step.copy_(self.rope_cos[p:p + 1])
            sin_step.copy_(self.rope_sin[p:p + 1])
            cur = run_step().clone()
            outs.append(cur)
        return torch.cat(outs, dim=1)
