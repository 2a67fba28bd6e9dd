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

The reference ships no model code (it is a storage service); this is the dense-table consumer.
"""
from __future__ import annotations

import argparse
import json
import math
import os
from dataclasses import dataclass
from typing import Dict, List, Optional

import torch
import torch.nn.functional as F
from torch.autograd.function import once_differentiable

from .._lib import C
from ..ops import gemm as G
from ..ops.act8 import Act8, act8_wgrad
from ..ops.dense import DenseTable
from ..ops.linear import linear_act, linear_act_dgrad, linear_bias_grad
from ..ops.norm import layer_norm, layer_norm_act8, layer_norm_act8_backward, layer_norm_backward
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

    def n_params(self) -> int:
        d, f = self.d_model, self.d_ff
        return self.vocab * d + self.seq_len * d + self.n_layer * (3 * d * d + d * d + 2 * d * f + 9 * d + f) + 2 * d


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


class _ProjResidual(torch.autograd.Function):
    """x + proj(a) of a fused block, for attention's output ``a`` ``[B, heads, T, d / heads]``. Attention's own graph keeps ``a`` too (laid
    out by rows: a matrix of rows is a view of it)."""

    @staticmethod
    def forward(ctx, a, x, model, i):
        P, Gr = model.main.params, model.main.grads
        w = P[f"h{i}.proj.w"]
        ctx.w_grad, ctx.b_grad = Gr[f"h{i}.proj.w"], Gr[f"h{i}.proj.b"]
        ctx.save_for_backward(w, a)
        d = x.shape[-1]
        return linear_act(a.transpose(1, 2).reshape(-1, d), w, P[f"h{i}.proj.b"], residual=x.reshape(-1, d)).view(x.shape)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        w, a = ctx.saved_tensors
        B, heads, T, hd = a.shape
        dy2 = dy.reshape(-1, dy.shape[-1]).contiguous()
        G.gemm(dy2, a.transpose(1, 2).reshape(-1, heads * hd), a_mn=True, b_mn=True, out=ctx.w_grad, accumulate=True)
        linear_bias_grad(dy2, out=ctx.b_grad, accumulate=True)
        da = linear_act_dgrad(dy2, w, None)
        return da.view(B, T, heads, hd).transpose(1, 2), dy, None, None


class _MlpHalf(torch.autograd.Function):
    """x + out(gelu(fc(norm(x)))) of a fused block. The hidden layer is kept before GELU only, and formed again behind it."""

    @staticmethod
    def forward(ctx, x, model, i):
        P, Gr = model.main.params, model.main.grads
        x2 = x.reshape(-1, x.shape[-1])
        ctx.norm = _Norm(model, f"h{i}.ln2")
        keep = ctx.needs_input_grad[0]
        y, kept = ctx.norm.forward(x2, keep)
        w1, w2 = P[f"h{i}.fc.w"], P[f"h{i}.out.w"]
        if not keep:
            f = linear_act(y, w1, P[f"h{i}.fc.b"], act="gelu_tanh")
        else:
            f, h = linear_act(y, w1, P[f"h{i}.fc.b"], act="gelu_tanh", save="act8" if ctx.norm.bits == 8 else "bf16")
            ctx.grads = [Gr[f"h{i}.{name}"] for name in ("fc.w", "fc.b", "out.w", "out.b")]
            ctx.save_for_backward(w1, w2, *((h.q, h.e) if ctx.norm.bits == 8 else (h, None)), *kept)
        return linear_act(f, w2, P[f"h{i}.out.b"], residual=x2).view(x.shape)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        w1, w2, h, e, *kept = ctx.saved_tensors
        w1_grad, b1_grad, w2_grad, b2_grad = ctx.grads
        dy2 = dy.reshape(-1, dy.shape[-1]).contiguous()
        dh, f = linear_act_dgrad(dy2, w2, h if e is None else Act8(h, e, w1.shape[0]), act="gelu_tanh", recompute=True)
        del h, e
        G.gemm(dy2, f, a_mn=True, b_mn=True, out=w2_grad, accumulate=True)
        del f
        linear_bias_grad(dy2, out=b2_grad, accumulate=True)
        ctx.norm.wgrad(kept, dh, w1_grad, b1_grad)
        dx = ctx.norm.backward(kept, linear_act_dgrad(dh, w1, None), residual_grad=dy2)
        return dx.view(dy.shape), None, None


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
        self.cfg = cfg
        self.group = group
        self.world, self.rank = _dist_info(group)
        self.device = torch.device(device) if device is not None else torch.device("cuda", torch.cuda.current_device())
        d, f, L = cfg.d_model, cfg.d_ff, cfg.n_layer
        opt = dict(lr=cfg.lr, weight_decay=cfg.weight_decay, beta2=0.95)
        shapes: Dict[str, tuple] = {"wte": (cfg.vocab, d), "wpe": (cfg.seq_len, d), "lnf.g": (d,), "lnf.b": (d,)}
        for i in range(L):
            shapes.update({f"h{i}.ln1.g": (d,), f"h{i}.ln1.b": (d,), f"h{i}.qkv.b": (3 * d,), f"h{i}.proj.w": (d, d),
                           f"h{i}.proj.b": (d,), f"h{i}.ln2.g": (d,), f"h{i}.ln2.b": (d,), f"h{i}.fc.w": (f, d),
                           f"h{i}.fc.b": (f,), f"h{i}.out.w": (d, f), f"h{i}.out.b": (d,)})
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

    def forward(self, tokens: torch.Tensor, targets: Optional[torch.Tensor] = None):
        cfg = self.cfg
        B, T = tokens.shape
        lv = self._leaves
        x = F.embedding(tokens, lv["wte"]) + lv["wpe"][:T]
        for i in range(cfg.n_layer):
            if cfg.fused:
                qkv, x = _NormedQkv.apply(x, self, i)
                a = self._attention(qkv, B, T)
                del qkv   # (a forward pass alone holds no more than it needs)
                x = _ProjResidual.apply(a, x, self, i)
                del a
                x = _MlpHalf.apply(x, self, i)
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
        """Collective, between steps: every dense table (values, optimizer slots, step count) under ``<uri>/table_<i>``."""
        from ..parallel import checkpoint
        torch.cuda.synchronize(self.device)
        for i, t in enumerate(self.tables):
            checkpoint.dump_dense(t, f"{uri.rstrip('/')}/table_{i}")

    def load_checkpoint(self, uri: str) -> None:
        """Collective, between steps; the checkpoint may come from a job with another number of ranks."""
        from ..parallel import checkpoint
        torch.cuda.synchronize(self.device)
        for i, t in enumerate(self.tables):
            checkpoint.load_dense(t, f"{uri.rstrip('/')}/table_{i}")


def _bench(args) -> None:
    import torch.distributed as dist
    world = int(os.environ.get("WORLD_SIZE", "1"))
    local = int(os.environ.get("LOCAL_RANK", "0"))
    torch.cuda.set_device(local)
    if world > 1:
        dist.init_process_group("nccl", device_id=torch.device("cuda", local))
    cfg = GPTConfig(n_layer=args.layers, fused=args.fused, act_bits=args.act_bits)
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
    ap.add_argument("--act-bits", type=int, default=16, choices=(16, 8), help="of what a fused block's norms and hidden layer keep for the backward pass")
    _bench(ap.parse_args())
