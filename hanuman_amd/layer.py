"""Device-resident MoE-layer forward for the measured workloads.

``DeviceLayer`` uploads one workload's inputs, packs its expert weights once
and runs the layer (router -> plan -> permute -> grouped SwiGLU -> combine)
entirely through ``libhanuman_moe.so``; ``forward`` is the step ``bench.py``
times and the GPU tests check.  With bf16 tokens and SwiGLU experts the
permutation is fused into the gate/up GEMM (``xs`` is then ``None``); with
fp8 experts on bf16 tokens the gate/up GEMM gathers from the per-token codes,
with mxfp4 experts from the tokens' 4-bit rows.
"""
from __future__ import annotations

import torch

from . import _lib
from . import kernels as K
from .workloads import Inputs, Workload

_TORCH_DT = {"bf16": torch.bfloat16, "f32": torch.float32}


class DeviceLayer:
    def __init__(self, inp: Inputs, device: str | torch.device = "cuda",
                 fused_ffn: bool | None = None):
        wl: Workload = inp.wl
        if wl.expert_dtype not in ("bf16", "fp8", "f32", "mxfp4"):
            raise NotImplementedError(f"{wl.name}: expert dtype {wl.expert_dtype} is not built")
        self.wl = wl
        self.fp8 = wl.expert_dtype == "fp8"
        self.f32 = wl.expert_dtype == "f32"
        self.mxfp4 = wl.expert_dtype == "mxfp4"
        dev = torch.device(device)
        self.device = dev
        self.x = torch.from_numpy(inp.x).to(dev, _TORCH_DT[wl.x_dtype]).contiguous()
        self.logits_in = None
        self.router_w = None
        if wl.router_from_logits:
            self.logits_in = torch.from_numpy(inp.logits).to(dev).contiguous()
        else:
            self.router_w = torch.from_numpy(inp.router).to(dev, _TORCH_DT[wl.router_w_dtype]).contiguous()
        self.mode = _lib.ROUTE_SOFTMAX if wl.routing == "softmax" else _lib.ROUTE_SIGMOID_BIAS
        self.capacity = wl.capacity
        self.w_gate_up = None
        self.w_down = None
        self.w_gate_up_scale = None
        self.w_down_scale = None
        self.w_gate_up_exp = self.w_down_exp = None
        self.w_gate = self.w_up = self.w_down_f32 = None
        if wl.expert == "swiglu" and self.f32:
            # float32 compute: the masters as they are
            self.w_gate = torch.from_numpy(inp.w_gate).to(dev).contiguous()
            self.w_up = torch.from_numpy(inp.w_up).to(dev).contiguous()
            self.w_down_f32 = torch.from_numpy(inp.w_down).to(dev).contiguous()
        elif wl.expert == "swiglu":
            wg = torch.from_numpy(inp.w_gate).to(dev)
            wu = torch.from_numpy(inp.w_up).to(dev)
            if self.fp8:
                self.w_gate_up, self.w_gate_up_scale = K.pack_fp8_gate_up(wg, wu)
            elif self.mxfp4:
                self.w_gate_up, self.w_gate_up_exp = K.pack_mxfp4_gate_up(wg, wu)
            else:
                self.w_gate_up = K.pack_gate_up(wg, wu)
            del wg, wu
            wd = torch.from_numpy(inp.w_down).to(dev)
            if self.fp8:
                self.w_down, self.w_down_scale = K.pack_fp8_down(wd)
            elif self.mxfp4:
                self.w_down, self.w_down_exp = K.pack_mxfp4_down(wd)
            else:
                self.w_down = K.pack_down(wd)
            del wd
        # bf16 SwiGLU experts on bf16 tokens: the gate/up GEMM gathers its rows
        # from x itself (hmoe_grouped_gate_up_gather), no dispatched copy.
        self.fused_dispatch = (wl.expert == "swiglu" and not self.fp8 and not self.mxfp4
                               and self.x.dtype == torch.bfloat16)
        # fp8 experts on bf16 tokens: x is quantised per token and the gate/up
        # GEMM gathers from its codes (hmoe_grouped_gate_up_fp8_gather).
        self.fp8_gather = (wl.expert == "swiglu" and self.fp8
                           and self.x.dtype == torch.bfloat16)
        ws = int(_lib.lib().hmoe_plan_workspace_bytes(wl.tokens, wl.top_k, wl.n_experts))
        self.workspace = torch.empty(max(ws, 1), dtype=torch.uint8, device=dev)
        # fused_ffn=True: the gathered gate/up GEMM and the down GEMM in one
        # persistent launch (hmoe_grouped_swiglu_fused) where its shape rules
        # hold.  Off by default: measured end to end it is within noise of the
        # two launches at the full bf16 workload and ~2 % slower at the skewed
        # one (the per-XCD split of whole m-tiles leaves up to one m-tile of
        # imbalance, about what the two launches' tails cost).
        can_fuse = (self.fused_dispatch and wl.d_model % 256 == 0 and wl.d_ff % 128 == 0
                    and wl.d_ff >= 256)
        self.fused_ffn = bool(fused_ffn) and can_fuse
        self.fused_ws = None
        if self.fused_ffn:
            rc = K.rows_cap(wl.tokens, wl.top_k, wl.n_experts, self.capacity)
            n = int(_lib.lib().hmoe_grouped_swiglu_fused_workspace_bytes(rc, wl.n_experts))
            self.fused_ws = torch.zeros(max(n, 64), dtype=torch.uint8, device=dev)
        self.out_dtype = _TORCH_DT[wl.out_dtype]

    # ---- stages (each enqueues on the current stream) ----------------------
    def route(self):
        wl = self.wl
        if self.logits_in is not None:
            top_idx, gates = K.router_from_logits(self.logits_in, None, wl.top_k, self.mode)
            return self.logits_in, top_idx, gates
        return K.router(self.x, self.router_w, None, wl.top_k, self.mode)

    def route_quant(self):
        """The router and, for fp8 experts gathering from per-token codes and for
        mxfp4 experts on bf16 tokens, x's quantisation in the same launch
        (``hmoe_router_quant_fp8``, ``hmoe_router_quant_mxfp4``: it runs beside the
        router's float64 MFMA chains).  Returns (logits, top_idx, gates, (x_q,
        x_scale) or None)."""
        wl = self.wl
        if self.fp8_gather and self.logits_in is None:
            logits, top_idx, gates, x_q, x_s = K.router_quant_fp8(self.x, self.router_w, None,
                                                                   wl.top_k, self.mode)
            return logits, top_idx, gates, (x_q, x_s)
        if self.mxfp4 and wl.expert == "swiglu" and self.x.dtype == torch.bfloat16 and self.logits_in is None:
            logits, top_idx, gates, x_q, x_e = K.router_quant_mxfp4(self.x, self.router_w, None,
                                                                     wl.top_k, self.mode)
            return logits, top_idx, gates, (x_q, x_e)
        return (*self.route(), None)

    def experts_fp8(self, plan, xq=None):
        """e4m3 dispatch and expert GEMMs: (xs_q, xs_scale, h_q, h_exp, ys).
        With bf16 tokens x is quantised per token and the gate/up GEMM gathers
        its rows from the codes (``xs_q``/``xs_scale`` are then per token,
        ``[T, D]``/``[T]``); otherwise they are the dispatched rows.  h leaves
        the gate/up GEMM block-scaled (codes ``h_q``, biased exponents
        ``h_exp`` per 32 columns) and the down GEMM's MFMA applies them.
        ``xq``: x's codes and scales when the router's launch made them."""
        if self.fp8_gather:
            xs_q, xs_s = xq if xq is not None else K.quantize_rows_fp8(self.x)
            h_q, h_e = K.grouped_gate_up_fp8_gather_qh(xs_q, xs_s, plan, self.w_gate_up,
                                                       self.w_gate_up_scale)
        else:
            xs_q, xs_s = K.permute_rows_fp8(self.x, plan)
            h_q, h_e = K.grouped_gate_up_fp8_qh(xs_q, xs_s, plan.offsets, self.w_gate_up,
                                                self.w_gate_up_scale)
        ys = K.grouped_down_fp8_mx(h_q, h_e, plan.offsets, self.w_down, self.w_down_scale)
        return xs_q, xs_s, h_q, h_e, ys

    def experts_mxfp4(self, plan, xq=None):
        """MXFP4 tokens and expert GEMMs: (x_q, x_exp, h_q, h_exp, ys), codes and biased
        exponents of the tokens and of h.  ``xq``: the tokens' when the router's launch
        made them."""
        x_q, x_e = xq if xq is not None else K.quantize_rows_mxfp4(self.x)
        h_q, h_e = K.grouped_gate_up_mxfp4_gather(x_q, x_e, plan, self.w_gate_up, self.w_gate_up_exp)
        ys = K.grouped_down_mxfp4(h_q, h_e, plan.offsets, self.w_down, self.w_down_exp)
        return x_q, x_e, h_q, h_e, ys

    def forward(self) -> dict:
        wl = self.wl
        logits, top_idx, gates, xq = self.route_quant()
        plan = K.dispatch_plan(top_idx, wl.n_experts, self.capacity, self.workspace)
        extra = {}
        h = None
        if self.fp8:
            xs, xs_s, h_q, h_e, ys = self.experts_fp8(plan, xq)
            extra = {"xs_scale": xs_s, "h_q": h_q, "h_exp": h_e,
                     "xs_per_token": self.fp8_gather}
        elif self.mxfp4 and wl.expert == "swiglu":
            x_q, x_e, h_q, h_e, ys = self.experts_mxfp4(plan, xq)
            xs = None
            extra = {"x_q": x_q, "x_exp": x_e, "h_q": h_q, "h_exp": h_e}
        elif self.f32:
            xs = K.permute_rows(self.x, plan, torch.float32)
            h = K.grouped_gate_up_f32(xs, plan.offsets, self.w_gate, self.w_up)
            ys = K.grouped_down_f32(h, plan.offsets, self.w_down_f32)
        elif self.fused_ffn:
            xs = None
            h, ys, ws = K.grouped_swiglu_fused(self.x, plan, self.w_gate_up, self.w_down,
                                               self.fused_ws)
            # a down tile whose bounded wait gave up computed from an
            # incomplete h: refuse the result (reading the status synchronises,
            # so not while a graph is being captured)
            if not torch.cuda.is_current_stream_capturing() and K.fused_status(ws) != 0:
                raise RuntimeError("grouped_swiglu_fused: a down tile's wait for its gate/up "
                                   "tiles timed out; h and ys are not valid")
        elif self.fused_dispatch:
            xs = None
            h = K.grouped_gate_up_gather(self.x, plan, self.w_gate_up)
            ys = K.grouped_down(h, plan.offsets, self.w_down)
        else:
            xs = K.permute_rows(self.x, plan, torch.bfloat16)
            if wl.expert == "identity":
                ys = xs
            else:
                h = K.grouped_gate_up(xs, plan.offsets, self.w_gate_up)
                ys = K.grouped_down(h, plan.offsets, self.w_down)
        out = K.combine(ys, plan, gates, None, self.out_dtype)
        return {"logits": logits, "top_idx": top_idx, "gates": gates, "plan": plan, "xs": xs,
                "h": h, "ys": ys, "out": out, **extra}
