"""GPT-style decoder trained with its dense parameters on the parameter server.

Config 4 of the benchmark: 24 layers, d_model 2048, 16 heads, FFN 8192, vocab 50304, sequence 2048, bf16,
data parallel over the GPUs of one box. Every linear layer runs on the tcgen05 GEMM (forward, dgrad,
wgrad accumulating in fp32 straight into the dense table's gradient buffer). Dense push = the fused
reduce-scatter + sharded AdamW kernel. Dense pull of the QKV weights = the all-gather fused into the QKV
GEMM (``ops.gemm.ag_linear``): each layer's ``W_qkv`` is its own table with ``scatter_peers=False``, so
after a push only the owner's rows are current and the first consumer gathers the rest over NVLink while
it already multiplies the local rows. Attention itself is model code, not a parameter-server path: it uses
``torch.nn.functional.scaled_dot_product_attention``; layer norm and GELU are torch ops, or, with ``GPTConfig(fused=True)``,
the block operators of this package: ``ops.norm`` for layer norm, ``ops.linear`` for linear layers with bias, GELU and residual
in their epilogue. ``act_bits=8`` keeps the norms' rows and the hidden layer before GELU in 8 bits for the backward pass
(``ops.act8``); what attention itself keeps (q, k, v and its output, which the projection's weight gradient reads too) stays in 16.
Fused blocks may have a gated hidden layer in place of GELU's (``gated=True``: ``ops.gated``, twice the first layer's weight), rotary positions in
place of the table of learned ones (``rotary=True``: ``ops.rotary``, on q and k where the QKV product left them), and dropout behind the
embedding and both halves of a block while training (``dropout=p``: ``ops.dropout``, in the epilogue of the second linear layer of each half).

The reference ships no model code (it is a storage service); this is the dense-table consumer.
"""
from __future__ import annotations

import argparse
import json
import math
import os
import weakref
from dataclasses import dataclass
from typing import Dict, List, Optional

import torch
import torch.nn.functional as F
from torch.autograd.function import once_differentiable

from .._lib import C
from ..ops import gemm as G
from ..ops.act8 import Act8, act8_wgrad
from ..ops.dense import DenseTable
from ..ops.dropout import drop_args, dropout, dropout_backward
from ..ops.gated import gated_linear, gated_linear_dgrad
from ..ops.linear import linear_act, linear_act_dgrad, linear_bias_grad
from ..ops.norm import layer_norm, layer_norm_act8, layer_norm_act8_backward, layer_norm_backward
from ..ops.rotary import rotary, rotary_backward, rotary_frequencies
from ..ops.sparse import _dist_info, _stream


@dataclass
class GPTConfig:
    n_layer: int = 24
    d_model: int = 2048
    n_head: int = 16
    d_ff: int = 8192
    vocab: int = 50304
    seq_len: int = 2048
    lr: float = 3e-4
    weight_decay: float = 0.1
    fused: bool = False   # blocks on ops.norm / ops.linear instead of torch ops around the GEMM
    act_bits: int = 16    # of what a fused block's norms and hidden layer keep for the backward pass: 16 or 8
    gated: bool = False   # fused blocks: silu(g) * u in place of gelu(h) in the hidden layer
    rotary: bool = False  # fused blocks: rotary positions of q and k in place of learned positions
    rotary_base: float = 10000.0
    dropout: float = 0.0  # fused blocks: behind the embedding and both halves of a block, in passes that train

    def n_params(self) -> int:
        d, f = self.d_model, self.d_ff
        hidden = 2 * f if self.gated else f
        return (self.vocab * d + (0 if self.rotary else self.seq_len * d)
                + self.n_layer * (3 * d * d + d * d + d * hidden + d * f + 9 * d + hidden) + 2 * d)


class _PSLinear(torch.autograd.Function):
    """y = x W^T + b on the tcgen05 GEMM; the weight / bias gradients are accumulated into the dense table's
    fp32 gradient views instead of being returned to autograd."""

    @staticmethod
    def forward(ctx, x, w, b, w_grad, b_grad, ag_table, ag_name):
        x2 = x.reshape(-1, x.shape[-1])
        if ag_table is not None:
            y = G.ag_linear(x2, ag_table, ag_name, bias=b)
        else:
            y = G.gemm(x2, w, bias=b)
        ctx.save_for_backward(x2, w)
        ctx.w_grad, ctx.b_grad = w_grad, b_grad
        ctx.shape = x.shape
        return y.view(*x.shape[:-1], w.shape[0])

    @staticmethod
    def backward(ctx, dy):
        x2, w = ctx.saved_tensors
        dy2 = dy.reshape(-1, dy.shape[-1]).contiguous()
        dx = G.gemm(dy2, w, b_mn=True)
        G.gemm(dy2, x2, a_mn=True, b_mn=True, out=ctx.w_grad, accumulate=True)
        if ctx.b_grad is not None:
            rc = C.bias_grad(dy2.data_ptr(), dy2.stride(0), dy2.shape[0], dy2.shape[1], ctx.b_grad.data_ptr(), _stream())
            if rc != 0:
                raise RuntimeError(f"bias_grad failed: {rc}")
        return dx.view(ctx.shape), None, None, None, None, None, None


class _Norm:
    """A layer norm of a fused model: its parameters, their gradients' places in the dense table, and its two passes. What lies between
    these (``kept``) is autograd's to save."""

    def __init__(self, model: "GPT", name: str):
        P, Gr = model.main.params, model.main.grads
        self.g, self.b = P[f"{name}.g"].detach(), P[f"{name}.b"].detach()
        self.g_grad, self.b_grad = Gr[f"{name}.g"], Gr[f"{name}.b"]
        self.bits = model.cfg.act_bits

    def forward(self, x: torch.Tensor, keep: bool):
        """(y, kept); nothing is kept where no backward pass can follow."""
        if not keep:
            return layer_norm(x, self.g, self.b)[0], ()
        if self.bits == 8:
            y, xhat8, rstd = layer_norm_act8(x, self.g, self.b)
            return y, (self.g, self.b, xhat8.q, xhat8.e, rstd)
        y, mean, rstd = layer_norm(x, self.g, self.b)
        return y, (self.g, self.b, x, mean, rstd, y)

    def backward(self, kept, dy: torch.Tensor, residual_grad: Optional[torch.Tensor] = None) -> torch.Tensor:
        kw = dict(residual_grad=residual_grad, weight_grad=self.g_grad, bias_grad=self.b_grad, accumulate=True)
        if self.bits == 8:
            g, _, q, e, rstd = kept
            return layer_norm_act8_backward(dy, Act8(q, e, g.numel()), g, rstd, **kw)[0]
        g, _, x, mean, rstd, _ = kept
        return layer_norm_backward(dy, x, g, mean, rstd, **kw)[0]

    def wgrad(self, kept, dy: torch.Tensor, w_grad: torch.Tensor, b_grad: torch.Tensor) -> None:
        """Gradients of the linear layer that took ``y``."""
        if self.bits == 8:
            g, b, q, e, _ = kept
            db = linear_bias_grad(dy)
            act8_wgrad(dy, Act8(q, e, g.numel()), weight=g, bias=b, dy_sum=db, out=w_grad, accumulate=True)
            b_grad.add_(db)
        else:
            G.gemm(dy, kept[-1], a_mn=True, b_mn=True, out=w_grad, accumulate=True)
            linear_bias_grad(dy, out=b_grad, accumulate=True)


class _NormedQkv(torch.autograd.Function):
    """(qkv(norm(x)), x) of a fused block: x goes on to the residual sum through here, so that its gradient joins the norm's where that is
    formed. Gradients of the parameters go to the dense tables."""

    @staticmethod
    def forward(ctx, x, model, i):
        P, table = model.main.params, model.qkv[i]
        ctx.norm = _Norm(model, f"h{i}.ln1")
        y, kept = ctx.norm.forward(x.reshape(-1, x.shape[-1]), ctx.needs_input_grad[0])
        if table is not None:
            w, ctx.w_grad = table.params["w"], table.grads["w"]
            qkv = G.ag_linear(y, table, "w", bias=P[f"h{i}.qkv.b"])
        else:
            w, ctx.w_grad = P[f"h{i}.qkv.w"], model.main.grads[f"h{i}.qkv.w"]
            qkv = linear_act(y, w, P[f"h{i}.qkv.b"])
        ctx.b_grad = model.main.grads[f"h{i}.qkv.b"]
        ctx.save_for_backward(w, *kept)
        return qkv, x

    @staticmethod
    @once_differentiable
    def backward(ctx, dqkv, dx):
        w, *kept = ctx.saved_tensors
        dqkv = dqkv.contiguous()
        ctx.norm.wgrad(kept, dqkv, ctx.w_grad, ctx.b_grad)
        dx2 = ctx.norm.backward(kept, linear_act_dgrad(dqkv, w, None), residual_grad=dx.reshape(-1, dx.shape[-1]))
        return dx2.view(dx.shape), None, None


class _NormedHeads(torch.autograd.Function):
    """(q, k, v, x) of a fused block with rotary positions: :class:`_NormedQkv`, with q and k turned where the product left them, as heads
    ``[B, heads, T, d / heads]``. Their gradients meet in one matrix again on the way back."""

    @staticmethod
    def _heads(qkv, model, B, T):
        H = model.cfg.n_head
        return qkv.view(B, T, 3, H, model.cfg.d_model // H).unbind(2)

    @staticmethod
    def forward(ctx, x, model, i):
        qkv, _ = _NormedQkv.forward(ctx, x, model, i)
        ctx.model = model
        q, k, v = _NormedHeads._heads(qkv, model, *x.shape[:2])
        rotary(q, k, model.freqs, out_q=q, out_k=k)
        return q.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2), x

    @staticmethod
    @once_differentiable
    def backward(ctx, dq, dk, dv, dx):
        B, T, d = dx.shape
        dqkv = dq.new_empty((B * T, 3 * d))
        q, k, v = _NormedHeads._heads(dqkv, ctx.model, B, T)
        rotary_backward(dq.transpose(1, 2), dk.transpose(1, 2), ctx.model.freqs, out_q=q, out_k=k)
        v.copy_(dv.transpose(1, 2))
        return _NormedQkv.backward(ctx, dqkv, dx)


class _DropPass:
    """A forward pass that drops values. ``number`` is another one for every pass, and for a pass that is computed again the one it had, as
    ``seed`` is. ``alone``: no other pass whose graph lives began with torch's generator in the same state."""

    __slots__ = ("number", "seed", "alone", "__weakref__")

    def __init__(self, number: int, seed):
        self.number, self.seed, self.alone = number, seed, True


class _Dropout(torch.autograd.Function):
    """Dropout with ``drop`` = (p, seed, offset); what it dropped is formed again on the way back. ``of``, the :class:`_DropPass` that it begins,
    lives as long as the pass's graph."""

    @staticmethod
    def forward(ctx, x, drop, of):
        ctx.drop, ctx.of = drop, of
        return dropout(x, *drop)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        return dropout_backward(dy, *ctx.drop), None, None


class _ProjResidual(torch.autograd.Function):
    """x + dropout(proj(a)) of a fused block, for attention's output ``a`` ``[B, heads, T, d / heads]``. Attention's own graph keeps ``a`` too
    (laid out by rows: a matrix of rows is a view of it)."""

    @staticmethod
    def forward(ctx, a, x, model, i, drop):
        P, Gr = model.main.params, model.main.grads
        w = P[f"h{i}.proj.w"]
        ctx.w_grad, ctx.b_grad = Gr[f"h{i}.proj.w"], Gr[f"h{i}.proj.b"]
        ctx.save_for_backward(w, a)
        ctx.drop = drop
        d = x.shape[-1]
        return linear_act(a.transpose(1, 2).reshape(-1, d), w, P[f"h{i}.proj.b"], residual=x.reshape(-1, d), dropout=drop).view(x.shape)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        w, a = ctx.saved_tensors
        B, heads, T, hd = a.shape
        dz = _before_dropout(dy.reshape(-1, dy.shape[-1]).contiguous(), ctx.drop)
        G.gemm(dz, a.transpose(1, 2).reshape(-1, heads * hd), a_mn=True, b_mn=True, out=ctx.w_grad, accumulate=True)
        linear_bias_grad(dz, out=ctx.b_grad, accumulate=True)
        da = linear_act_dgrad(dz, w, None)
        return da.view(B, T, heads, hd).transpose(1, 2), dy, None, None, None


def _before_dropout(dy, drop):
    return dy if drop is None else dropout_backward(dy, *drop)


class _MlpHalf(torch.autograd.Function):
    """x + dropout(out(gelu(fc(norm(x))))) of a fused block, or of one whose hidden layer is gated, silu(g) * u with [g | u] = fc(norm(x)). The
    hidden layer is kept before its activation only, and formed again behind it."""

    @staticmethod
    def forward(ctx, x, model, i, drop):
        P, Gr = model.main.params, model.main.grads
        x2 = x.reshape(-1, x.shape[-1])
        ctx.norm = _Norm(model, f"h{i}.ln2")
        keep = ctx.needs_input_grad[0]
        y, kept = ctx.norm.forward(x2, keep)
        w1, w2 = P[f"h{i}.fc.w"], P[f"h{i}.out.w"]
        hidden, act = (gated_linear, "silu") if model.cfg.gated else (linear_act, "gelu_tanh")
        if not keep:
            f = hidden(y, w1, P[f"h{i}.fc.b"], act=act)
        else:
            f, h = hidden(y, w1, P[f"h{i}.fc.b"], act=act, save="act8" if ctx.norm.bits == 8 else "bf16")
            ctx.gated, ctx.drop = model.cfg.gated, drop
            ctx.grads = [Gr[f"h{i}.{name}"] for name in ("fc.w", "fc.b", "out.w", "out.b")]
            # (in 8 bits: whole numbers and exponents of the hidden layer, or of both factors of a gated one)
            saved = (h,) if ctx.norm.bits != 8 else (h[0].q, h[0].e, h[1].q, h[1].e) if ctx.gated else (h.q, h.e)
            ctx.n_hidden = len(saved)
            ctx.save_for_backward(w1, w2, *saved, *kept)
        return linear_act(f, w2, P[f"h{i}.out.b"], residual=x2, dropout=drop).view(x.shape)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        w1, w2, *rest = ctx.saved_tensors
        h, kept = rest[:ctx.n_hidden], rest[ctx.n_hidden:]
        del rest
        w1_grad, b1_grad, w2_grad, b2_grad = ctx.grads
        dy2 = dy.reshape(-1, dy.shape[-1]).contiguous()
        dz = _before_dropout(dy2, ctx.drop)
        if ctx.gated:
            F2 = w2.shape[1]
            dh, f = gated_linear_dgrad(dz, w2, h[0] if len(h) == 1 else (Act8(h[0], h[1], F2), Act8(h[2], h[3], F2)), act="silu", recompute=True)
        else:
            dh, f = linear_act_dgrad(dz, w2, h[0] if len(h) == 1 else Act8(h[0], h[1], w1.shape[0]), act="gelu_tanh", recompute=True)
        del h
        G.gemm(dz, f, a_mn=True, b_mn=True, out=w2_grad, accumulate=True)
        del f
        linear_bias_grad(dz, out=b2_grad, accumulate=True)
        del dz
        ctx.norm.wgrad(kept, dh, w1_grad, b1_grad)
        dx = ctx.norm.backward(kept, linear_act_dgrad(dh, w1, None), residual_grad=dy2)
        return dx.view(dy.shape), None, None, None


class _FinalNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, model):
        ctx.norm = _Norm(model, "lnf")
        y, kept = ctx.norm.forward(x.reshape(-1, x.shape[-1]), ctx.needs_input_grad[0])
        ctx.save_for_backward(*kept)
        return y.view(x.shape)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        return ctx.norm.backward(ctx.saved_tensors, dy.reshape(-1, dy.shape[-1])).view(dy.shape), None


class GPT:
    def __init__(self, cfg: GPTConfig, *, device=None, group=None, seed: int = 0, fuse_qkv_gather: bool = True):
        if cfg.act_bits not in (8, 16) or (cfg.act_bits == 8 and not cfg.fused):
            raise ValueError("GPTConfig: act_bits is 16, or 8 with fused=True")
        if (cfg.gated or cfg.rotary or cfg.dropout) and not cfg.fused:
            raise ValueError("GPTConfig: gated, rotary and dropout need fused=True")
        if cfg.rotary and cfg.d_model // cfg.n_head % 2:
            raise ValueError(f"GPTConfig: rotary needs heads of an even number of values, not {cfg.d_model // cfg.n_head}")
        drop_args(cfg.dropout, 0, 0, -1, "GPTConfig: dropout")
        self.cfg = cfg
        self.group = group
        self.world, self.rank = _dist_info(group)
        self.device = torch.device(device) if device is not None else torch.device("cuda", torch.cuda.current_device())
        d, f, L = cfg.d_model, cfg.d_ff, cfg.n_layer
        opt = dict(lr=cfg.lr, weight_decay=cfg.weight_decay, beta2=0.95)
        shapes: Dict[str, tuple] = {"wte": (cfg.vocab, d), "wpe": (cfg.seq_len, d), "lnf.g": (d,), "lnf.b": (d,)}
        if cfg.rotary:
            del shapes["wpe"]
            self.freqs = rotary_frequencies(d // cfg.n_head, cfg.rotary_base, device=self.device)[0]
        # every rank drops values of its own; `drop_passes` counts the forward passes that did, so that each of them draws anew
        self.drop_seed, self.drop_passes = (seed << 16) + self.rank & 0xFFFFFFFFFFFFFFFF, 0
        self._drop_known = weakref.WeakValueDictionary()   # by what they drew of torch's generator: the passes whose graphs live
        self._replays = torch.zeros((), dtype=torch.int64, device=self.device) if cfg.dropout and self.device.type == "cuda" else None
        h = 2 * f if cfg.gated else f   # outputs of the hidden layer's product
        for i in range(L):
            shapes.update({f"h{i}.ln1.g": (d,), f"h{i}.ln1.b": (d,), f"h{i}.qkv.b": (3 * d,), f"h{i}.proj.w": (d, d),
                           f"h{i}.proj.b": (d,), f"h{i}.ln2.g": (d,), f"h{i}.ln2.b": (d,), f"h{i}.fc.w": (h, d),
                           f"h{i}.fc.b": (h,), f"h{i}.out.w": (d, f), f"h{i}.out.b": (d,)})
        # the QKV weights can be gathered lazily by their consumer: one table per layer, rows sharded by rank
        self.lazy_qkv = fuse_qkv_gather and self.world > 1 and (3 * d) % (256 * self.world) == 0
        if not self.lazy_qkv:
            for i in range(L):
                shapes[f"h{i}.qkv.w"] = (3 * d, d)
        self.main = DenseTable(shapes, "adamw", opt, grad_dtype=torch.float32, device=self.device, group=group)
        self.qkv: List[Optional[DenseTable]] = []
        for i in range(L):
            self.qkv.append(DenseTable({"w": (3 * d, d)}, "adamw", opt, grad_dtype=torch.float32, device=self.device, group=group,
                                       scatter_peers=False) if self.lazy_qkv else None)
        gen = torch.Generator().manual_seed(seed)
        init = {}
        for name, shape in shapes.items():
            if name.endswith(".g"):
                init[name] = torch.ones(shape)
            elif name.endswith(".b"):
                init[name] = torch.zeros(shape)
            else:
                std = 0.02 / math.sqrt(2 * L) if (".proj.w" in name or ".out.w" in name) else 0.02
                init[name] = torch.randn(shape, generator=gen) * std
        self.main.load(init)
        for i, t in enumerate(self.qkv):
            if t is not None:
                t.load({"w": torch.randn((3 * d, d), generator=gen) * 0.02})
        # small parameters go through autograd as leaves that alias the table; their .grad is folded in later
        self._leaves = {}
        for name in shapes:
            if name in ("wte", "wpe") or (not cfg.fused and (".ln" in name or name.startswith("lnf."))):
                self._leaves[name] = self.main.params[name].requires_grad_(True)
        self.tables = [self.main] + [t for t in self.qkv if t is not None]

    # ------------------------------------------------------------------------------------------
    def _linear(self, x, wname, bname, ag_table=None):
        P, Gd = self.main.params, self.main.grads
        if ag_table is not None:
            return _PSLinear.apply(x, ag_table.params["w"], P[bname], ag_table.grads["w"], Gd[bname], ag_table, "w")
        return _PSLinear.apply(x, P[wname], P[bname], Gd[wname], Gd[bname], None, None)

    def _attention(self, qkv: torch.Tensor, B: int, T: int) -> torch.Tensor:
        q, k, v = qkv.view(B, T, 3, self.cfg.n_head, self.cfg.d_model // self.cfg.n_head).permute(2, 0, 3, 1, 4)
        return F.scaled_dot_product_attention(q, k, v, is_causal=True)

    def _pass_seed(self):
        """The seed of a pass. While a graph is captured it is one in memory, another at every replay (``2^40`` on, past those of other ranks),
        which the pass's backward pass reads, too."""
        if self._replays is None or not torch.cuda.is_current_stream_capturing():
            return self.drop_seed
        return self._replays.add_(1 << 40) + (self.drop_seed - (self.drop_seed >> 63 << 64))   # (as a number with a sign)

    def _drop_pass(self) -> _DropPass:
        """A new pass that drops values, or the one that is being computed again: recomputation (``torch.utils.checkpoint``) runs ``forward``
        once more inside the backward pass, and puts torch's generators back to where they were, so that the number which every pass draws of
        the CPU's tells which one it is."""
        drawn = int(torch.empty((), dtype=torch.int64, device="cpu").random_())
        known = self._drop_known.get(drawn)
        if torch._C._current_graph_task_id() == -1:   # not inside a backward pass
            one = self._drop_known[drawn] = _DropPass(self.drop_passes, self._pass_seed())
            self.drop_passes += 1
            if known is not None:
                one.alone = known.alone = False
            return one
        if known is None or not known.alone:
            raise RuntimeError("GPT: a pass with dropout that is recomputed inside a backward pass finds its masks only where torch.utils.checkpoint has "
                               "use_reentrant=False and preserve_rng_state=True, and torch's generators were not seeded alike ahead of several passes")
        return known

    def forward(self, tokens: torch.Tensor, targets: Optional[torch.Tensor] = None, *, drop: Optional[bool] = None):
        """``(logits, loss)``; without ``targets`` the loss is None. ``drop``: whether the pass has the dropout of the model's configuration; if
        it is not said, a pass with targets and gradients has it."""
        cfg = self.cfg
        B, T = tokens.shape
        lv = self._leaves
        x = F.embedding(tokens, lv["wte"])
        if not cfg.rotary:
            x = x + lv["wpe"][:T]
        drops = [None] * (2 * cfg.n_layer + 1)
        if drop is None:
            drop = targets is not None and torch.is_grad_enabled()
        if cfg.dropout and drop:
            of = self._drop_pass()
            drops = [(cfg.dropout, of.seed, (of.number << 16) + site) for site in range(2 * cfg.n_layer + 1)]
            x = _Dropout.apply(x, drops[-1], of)
        for i in range(cfg.n_layer):
            if cfg.fused:
                if cfg.rotary:
                    q, k, v, x = _NormedHeads.apply(x, self, i)
                    a = F.scaled_dot_product_attention(q, k, v, is_causal=True)
                    del q, k, v
                else:
                    qkv, x = _NormedQkv.apply(x, self, i)
                    a = self._attention(qkv, B, T)
                    del qkv   # (a forward pass alone holds no more than it needs)
                x = _ProjResidual.apply(a, x, self, i, drops[2 * i])
                del a
                x = _MlpHalf.apply(x, self, i, drops[2 * i + 1])
                continue
            h = F.layer_norm(x, (cfg.d_model,), lv[f"h{i}.ln1.g"], lv[f"h{i}.ln1.b"])
            qkv = self._linear(h, f"h{i}.qkv.w", f"h{i}.qkv.b", self.qkv[i])
            a = self._attention(qkv, B, T)
            a = a.transpose(1, 2).reshape(B, T, cfg.d_model)
            x = x + self._linear(a, f"h{i}.proj.w", f"h{i}.proj.b")
            h = F.layer_norm(x, (cfg.d_model,), lv[f"h{i}.ln2.g"], lv[f"h{i}.ln2.b"])
            h = F.gelu(self._linear(h, f"h{i}.fc.w", f"h{i}.fc.b"), approximate="tanh")
            x = x + self._linear(h, f"h{i}.out.w", f"h{i}.out.b")
        x = _FinalNorm.apply(x, self) if cfg.fused else F.layer_norm(x, (cfg.d_model,), lv["lnf.g"], lv["lnf.b"])
        # tied output embedding: the GEMM's weight gradient and the embedding's gradient both land in wte's slot
        logits = _PSLinear.apply(x, self.main.params["wte"], None, self.main.grads["wte"], None, None, None)
        if targets is None:
            return logits, None
        loss = F.cross_entropy(logits.float().view(-1, cfg.vocab), targets.reshape(-1))
        return logits, loss

    def zero_grads(self) -> None:
        for t in self.tables:
            t.zero_grads()
        for p in self._leaves.values():
            p.grad = None

    def train_step(self, tokens: torch.Tensor, targets: torch.Tensor, micro_batches: int = 1) -> torch.Tensor:
        """One optimizer step on this rank's batch (split into ``micro_batches`` accumulation steps): forward,
        backward, then the collective dense push of every table."""
        self.zero_grads()
        total = torch.zeros((), device=self.device)
        for tk, tg in zip(tokens.chunk(micro_batches), targets.chunk(micro_batches)):
            _, loss = self.forward(tk, tg)
            (loss / micro_batches).backward()
            total += loss.detach() / micro_batches
        for name, p in self._leaves.items():
            if p.grad is not None:
                self.main.grads[name].add_(p.grad.float())
        for t in self.tables:
            t.push()
        return total

    def check(self) -> None:
        for t in self.tables:
            t.check()
        G.check_gemm_errors()

    def save_checkpoint(self, uri: str) -> None:
        """Collective, between steps: every dense table (values, optimizer slots, step count) under ``<uri>/table_<i>``, and what the next
        pass draws its dropout masks from in ``<uri>/dropout.json``."""
        from ..parallel import checkpoint
        self._settle()
        if self.rank == 0:   # (ahead of the tables, whose end all ranks wait for)
            folder = uri.split("?", 1)[0]
            if checkpoint._is_remote(folder):
                raise ValueError("GPT.save_checkpoint writes to a local directory")
            os.makedirs(folder, exist_ok=True)
            tmp = os.path.join(folder, ".dropout.json.tmp")
            with open(tmp, "w") as f:
                json.dump({"seed": int(self.drop_seed), "passes": int(self.drop_passes)}, f)
            os.replace(tmp, os.path.join(folder, "dropout.json"))
        for i, t in enumerate(self.tables):
            checkpoint.dump_dense(t, f"{uri.rstrip('/')}/table_{i}")

    def load_checkpoint(self, uri: str) -> None:
        """Collective, between steps; the checkpoint may come from a job with another number of ranks. Dropout goes on with the masks that the
        job which wrote it would draw next (``drop_seed`` and ``drop_passes`` stay as they are where the checkpoint does not hold them)."""
        from ..parallel import checkpoint
        self._settle()
        for i, t in enumerate(self.tables):
            checkpoint.load_dense(t, f"{uri.rstrip('/')}/table_{i}")
        at = os.path.join(uri.split("?", 1)[0], "dropout.json")
        if os.path.exists(at):
            with open(at) as f:
                kept = json.load(f)
            self.drop_seed, self.drop_passes = int(kept["seed"]) + self.rank & 0xFFFFFFFFFFFFFFFF, int(kept["passes"])   # (rank 0 wrote it)

    def _settle(self) -> None:
        if self.device.type == "cuda":
            torch.cuda.synchronize(self.device)


def _bench(args) -> None:
    import torch.distributed as dist
    world = int(os.environ.get("WORLD_SIZE", "1"))
    local = int(os.environ.get("LOCAL_RANK", "0"))
    torch.cuda.set_device(local)
    if world > 1:
        dist.init_process_group("nccl", device_id=torch.device("cuda", local))
    cfg = GPTConfig(n_layer=args.layers, d_ff=args.d_ff, fused=args.fused, act_bits=args.act_bits, gated=args.gated, rotary=args.rotary, dropout=args.dropout)
    model = GPT(cfg, fuse_qkv_gather=not args.no_fuse)
    B = args.seqs_per_gpu
    gen = torch.Generator().manual_seed(local)
    tok = torch.randint(0, cfg.vocab, (B, cfg.seq_len + 1), generator=gen).pin_memory()
    d_tok = torch.empty_like(tok, device="cuda")
    for _ in range(args.warmup):
        d_tok.copy_(tok, non_blocking=True)
        model.train_step(d_tok[:, :-1], d_tok[:, 1:], args.micro)
    model.check()
    e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    if world > 1:
        dist.barrier()
    torch.cuda.synchronize()
    e0.record()
    for _ in range(args.steps):
        d_tok.copy_(tok, non_blocking=True)
        loss = model.train_step(d_tok[:, :-1], d_tok[:, 1:], args.micro)
    e1.record()
    torch.cuda.synchronize()
    ms = e0.elapsed_time(e1) / args.steps
    if world > 1:
        t = torch.tensor([ms], device="cuda")
        dist.all_reduce(t, op=dist.ReduceOp.MAX)
        ms = float(t.item())
    model.check()
    tokens = B * cfg.seq_len * world
    flops = 6 * cfg.n_params() * tokens + 12 * cfg.n_layer * cfg.d_model * cfg.seq_len * tokens
    if local == 0:
        print(json.dumps({"metric": "gpt_tokens_per_sec", "value": tokens / (ms / 1e3), "n_gpus": world, "ms_per_step": ms,
                          "model_tflops_per_gpu": flops / (ms / 1e3) / 1e12 / world, "layers": cfg.n_layer,
                          "params": cfg.n_params(), "global_batch_seqs": B * world, "seq_len": cfg.seq_len,
                          "qkv_gather_fused": model.lazy_qkv, "blocks_fused": cfg.fused, "act_bits": cfg.act_bits,
                          "d_ff": cfg.d_ff, "gated": cfg.gated, "rotary": cfg.rotary, "dropout": cfg.dropout,
                          "peak_gb": torch.cuda.max_memory_allocated() / 1e9, "loss": float(loss.item())}))
    if world > 1:
        dist.destroy_process_group()


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description="GPT dense-path benchmark (config 4): python -m parameter_server_b200.models.gpt")
    ap.add_argument("--layers", type=int, default=24)
    ap.add_argument("--seqs-per-gpu", type=int, default=8)
    ap.add_argument("--micro", type=int, default=2)
    ap.add_argument("--steps", type=int, default=3)
    ap.add_argument("--warmup", type=int, default=2)
    ap.add_argument("--no-fuse", action="store_true", help="all-gather the QKV weights in the dense push instead of in the GEMM")
    ap.add_argument("--fused", action="store_true", help="blocks on ops.norm / ops.linear")
    ap.add_argument("--d-ff", type=int, default=8192, help="hidden values of a block's MLP")
    ap.add_argument("--gated", action="store_true", help="fused blocks: silu(g) * u in place of gelu(h)")
    ap.add_argument("--rotary", action="store_true", help="fused blocks: rotary positions in place of learned ones")
    ap.add_argument("--dropout", type=float, default=0.0, help="fused blocks: share of values dropped behind the embedding and both halves of a block")
    ap.add_argument("--act-bits", type=int, default=16, choices=(16, 8), help="of what a fused block's norms and hidden layer keep for the backward pass")
    _bench(ap.parse_args())
