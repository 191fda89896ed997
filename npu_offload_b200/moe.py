"""Host-side API of the B200 routed-expert MoE data plane (a thin layer over the C ABI).

* ``MoEDataPlane`` -- one context per GPU: expert tables resident in HBM, and the per-layer hot path
  ``forward(layer, hidden, logits) -> out`` (the surface of the reference engine's
  ``Model::moe_phase``, track2_opt/solar_engine/src/main.rs:149-209, and of ``Runtime._moe``,
  solar_hybrid/runtime.py:338-423).
* ``gpu_moe`` / ``set_threads`` -- drop-in replacements for ``cpu_moe_ext.cpu_moe`` /
  ``cpu_moe_ext.set_threads`` (solar_hybrid/cpu_moe.cpp:38-105): same arguments, same result
  layout, same error on H or F not a multiple of 32.

PyTorch only provides device memory and streams here; every computation runs in libmoe_dp.so.
"""
import ctypes
import importlib.util
import os
from typing import NamedTuple

import numpy as np
import torch

from . import _lib
from ._lib import (MOE_F_ACCUMULATE, MOE_F_HOST, MOE_F_SYNC, MOE_SCORING_SIGMOID, MOE_SCORING_SOFTMAX,
                   MoeConfig, check, lib)
from .build import binding_path

__all__ = ["MoEDataPlane", "Fp8", "Normed", "BalanceStats", "gpu_moe", "set_threads", "as_bf16"]

_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)  # (a torch without CUDA has none, and no GPU path)
_calls = None  # the module _torch_binding, from its first use on


class Fp8(NamedTuple):
    """e4m3 values with one fp32 scale for each 128 columns of one row, or of 128 rows; value = q * scale."""
    q: torch.Tensor      # [..., rows, cols] torch.float8_e4m3fn
    scale: torch.Tensor  # [..., ceil(rows / block_rows), ceil(cols / 128)] torch.float32


class Normed(NamedTuple):
    """What add_norm() gives."""
    y: "torch.Tensor | None"  # sum * rstd * weight, of out_dtype (None: not asked for)
    fp8: "Fp8 | None"         # the same in e4m3, a scale for each 128 columns of a row (None: not asked for)
    sum: torch.Tensor         # x + residual, of the residual's type; without a residual, x itself
    rstd: torch.Tensor        # [...] fp32: 1 / sqrt(mean sum^2 + eps)


class BalanceStats(NamedTuple):
    """What balance_loss() counted, as balance_loss_backward() takes it."""
    counts: torch.Tensor            # [B, E] int32: choices of each expert, per sequence
    tokens: torch.Tensor            # [B + 1] int32: tokens that count, and the number of sequences with any
    offsets: "torch.Tensor | None"  # the sequences and the mask they were counted with
    mask: "torch.Tensor | None"


def _vp(t):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


def as_bf16(a, device=None):
    """numpy uint16 (bf16 bits) or torch bf16 -> contiguous torch bf16 tensor (optionally moved)."""
    if isinstance(a, np.ndarray):
        assert a.dtype == np.uint16, a.dtype
        t = torch.from_numpy(np.ascontiguousarray(a).view(np.int16)).view(torch.bfloat16)
    else:
        t = a
        if t.dtype == torch.int16 or t.dtype == torch.uint16:
            t = t.view(torch.bfloat16)
        assert t.dtype == torch.bfloat16, t.dtype
    if device is not None:
        t = t.to(device, non_blocking=False)
    return t.contiguous()


def _as(a, dtype, device=None):
    t = torch.as_tensor(a) if not isinstance(a, torch.Tensor) else a
    t = t.to(dtype)
    if device is not None:
        t = t.to(device)
    return t.contiguous()


def _stream_ptr(stream, device):
    if stream is None:
        stream = torch.cuda.current_stream(device)
    return ctypes.c_void_p(stream.cuda_stream)


class MoEDataPlane:
    """Expert tables + routed-expert forward for ``n_layers`` MoE layers on one GPU.

    Expert-parallel use: pass ``ep_rank`` / ``ep_world`` (and optionally a ``shard_map`` of shape
    [n_layers, n_experts] giving each expert's owner rank); ``forward`` then returns this rank's
    partial sum over its local experts, which npu_offload_b200.parallel combines across ranks.
    """

    def __init__(self, hidden, inter, n_experts, top_k=8, n_layers=1, max_tokens=64, scoring="softmax", device=0,
                 ep_rank=0, ep_world=1, shard_map=None):
        self.H, self.F, self.E, self.K, self.L = int(hidden), int(inter), int(n_experts), int(top_k), int(n_layers)
        self.max_tokens = int(max_tokens)
        self.device = torch.device("cuda", device) if isinstance(device, int) else torch.device(device)
        if self.device.index is None:
            self.device = torch.device("cuda", 0)
        self._index = self.device.index
        self._plane = None
        self.scoring = scoring
        sc = {"softmax": MOE_SCORING_SOFTMAX, "sigmoid": MOE_SCORING_SIGMOID}[scoring]
        self._shard = None
        if shard_map is not None:
            self._shard = np.ascontiguousarray(np.asarray(shard_map, dtype=np.int32).reshape(-1))
        cfg = MoeConfig(self.H, self.F, self.E, self.K, self.L, self.max_tokens, sc, self.device.index or 0,
                        int(ep_rank), int(ep_world),
                        None if self._shard is None else self._shard.ctypes.data_as(ctypes.POINTER(ctypes.c_int32)))
        self.ep_rank, self.ep_world = int(ep_rank), int(ep_world)
        self.ep_attached = False
        h = ctypes.c_void_p()
        check(lib().moe_create(ctypes.byref(cfg), ctypes.byref(h)))
        self._h = h

    # ---- lifetime ----
    # ---- expert-parallel peer exchange (collective set-up; see parallel.attach_peers) ----
    def ep_export(self):
        """This rank's exchange-buffer handle record (bytes)."""
        from ._lib import MOE_EP_RECORD_BYTES
        buf = ctypes.create_string_buffer(MOE_EP_RECORD_BYTES)
        check(lib().moe_ep_export(self._h, buf, MOE_EP_RECORD_BYTES))
        return buf.raw

    def ep_import(self, records):
        """Map every rank's exchange buffer (records of all ranks, rank order, concatenated); from
        then on forward() returns the full combined output on every rank."""
        check(lib().moe_ep_import(self._h, records, self.ep_world))
        self.ep_attached = True

    def close(self):
        if getattr(self, "_h", None):
            lib().moe_destroy(self._h)
            self._h = self._plane = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def __enter__(self):
        return self

    def __exit__(self, *a):
        self.close()

    @property
    def handle(self):
        return self._h

    def owner(self, layer, expert):
        if self._shard is not None:
            return int(self._shard[layer * self.E + expert])
        return 0 if self.ep_world == 1 else expert % self.ep_world

    # ---- expert tables ----
    def load_expert(self, layer, expert, gate, up, down):
        """gate/up [F,H], down [H,F] bf16 (torch, host or device, or numpy uint16 bits)."""
        g, u, d = (as_bf16(a) for a in (gate, up, down))
        assert g.shape == (self.F, self.H) and u.shape == (self.F, self.H) and d.shape == (self.H, self.F)
        flags = 0 if g.is_cuda else MOE_F_HOST
        if not g.is_cuda:
            u, d = u.cpu(), d.cpu()
        else:
            u, d = u.to(g.device), d.to(g.device)
        check(lib().moe_load_expert_bf16(self._h, layer, expert, _vp(g), _vp(u), _vp(d), flags))

    def load_expert_q8(self, layer, expert, q, scales):
        """q int8 [3*F*H] in the ck_place_expert_q8 layout, scales fp32 [2F+H]."""
        qt = _as(q, torch.int8)
        st = _as(scales, torch.float32, qt.device)
        flags = 0 if qt.is_cuda else MOE_F_HOST
        check(lib().moe_load_expert_q8(self._h, layer, expert, _vp(qt), _vp(st), flags))

    def quantize_expert_q8(self, layer, expert):
        check(lib().moe_quantize_expert_q8(self._h, layer, expert))

    def evict_expert(self, layer, expert):
        """Frees the expert's HBM slot (MOE_OPT_LAYER_SLOTS tables); it reads as not loaded afterwards."""
        check(lib().moe_evict_expert(self._h, layer, expert))

    def _bias(self, bias, device=None):
        b = _as(bias, torch.float32, device)
        if b.numel() != self.E:
            raise ValueError(f"bias is {tuple(b.shape)}, the context has {self.E} experts")
        return b

    def expert_kind(self, layer, expert):
        return lib().moe_expert_kind(self._h, layer, expert)

    def set_bias(self, layer, bias):
        if bias is None:
            check(lib().moe_set_bias(self._h, layer, None, 0))
            return
        b = self._bias(bias)
        check(lib().moe_set_bias(self._h, layer, _vp(b), 0 if b.is_cuda else MOE_F_HOST))

    # ---- hot path ----
    def forward(self, layer, hidden, logits, out=None, return_topk=False, accumulate=False, stream=None, sync=False):
        """hidden [T,H] bf16, logits [T,E] fp32 (device tensors) -> out [T,H] fp32 on the device.

        Asynchronous on ``stream`` (default: torch's current stream) unless ``sync``."""
        x = as_bf16(hidden)
        lg = _as(logits, torch.float32)
        T = x.shape[0]
        assert x.is_cuda and lg.is_cuda and x.shape[1] == self.H and lg.shape == (T, self.E)
        if out is None:
            out = torch.empty(T, self.H, dtype=torch.float32, device=x.device)
        idx = w = None
        if return_topk:
            idx = torch.empty(T, self.K, dtype=torch.int32, device=x.device)
            w = torch.empty(T, self.K, dtype=torch.float32, device=x.device)
        flags = (MOE_F_ACCUMULATE if accumulate else 0) | (MOE_F_SYNC if sync else 0)
        check(lib().moe_forward(self._h, layer, T, _vp(x), _vp(lg), _vp(out), _vp(idx), _vp(w), flags,
                                _stream_ptr(stream, x.device)))
        return (out, idx, w) if return_topk else out

    def forward_layers(self, layers, hiddens, logits, outs, accumulate=False, stream=None, sync=False):
        """Several layer calls enqueued by one C call (moe_forward_layers): layer layers[i] on
        hiddens[i] [T,H] bf16 and logits[i] [T,E] fp32 into outs[i] [T,H] fp32, device tensors, in
        order."""
        n = len(layers)
        assert len(hiddens) == len(logits) == len(outs) == n
        T = hiddens[0].shape[0] if n else 0
        for x, lg, o in zip(hiddens, logits, outs):
            assert x.is_cuda and x.dtype == torch.bfloat16 and x.shape == (T, self.H)
            assert lg.is_cuda and lg.dtype == torch.float32 and lg.shape == (T, self.E)
            assert o.is_cuda and o.dtype == torch.float32 and o.shape == (T, self.H)
        la = (ctypes.c_int32 * max(n, 1))(*layers)
        xa = (ctypes.c_void_p * max(n, 1))(*[t.data_ptr() for t in hiddens])
        ga = (ctypes.c_void_p * max(n, 1))(*[t.data_ptr() for t in logits])
        oa = (ctypes.c_void_p * max(n, 1))(*[t.data_ptr() for t in outs])
        flags = (MOE_F_ACCUMULATE if accumulate else 0) | (MOE_F_SYNC if sync else 0)
        dev = hiddens[0].device if n else self.device
        check(lib().moe_forward_layers(self._h, n, la, T, xa, ga, oa, flags, _stream_ptr(stream, dev)))
        return outs

    # ---- the steps either side of the routed experts (one Solar MoE block, solar_engine/src/layer.rs:1-6) ----
    def load_shared(self, layer, gate=None, up=None, down=None, router=None):
        """Shared expert gate/up [Fs,H], down [H,Fs] and router weights [E,H] (bf16) of one layer.
        Fs may differ from the routed F (a context holding a slice of every routed expert's units
        still holds the whole shared expert); it is fixed by the first load."""
        from ._lib import MOE_OPT_SHARED_INTER
        ws = [None if a is None else as_bf16(a) for a in (gate, up, down, router)]
        on_dev = [w.is_cuda for w in ws if w is not None]
        dev = bool(on_dev) and on_dev[0]
        ws = [None if w is None else (w.to(self.device) if dev else w.cpu()) for w in ws]
        if ws[0] is not None:
            fs = ws[0].shape[0]
            assert ws[0].shape == (fs, self.H) and ws[1].shape == (fs, self.H) and ws[2].shape == (self.H, fs)
            if getattr(self, "_shared_inter", None) != fs:
                self.set_option(MOE_OPT_SHARED_INTER, fs)
                self._shared_inter = fs
        if ws[3] is not None:
            assert ws[3].shape == (self.E, self.H)
        check(lib().moe_load_shared(self._h, layer, *[_vp(w) for w in ws], 0 if dev else MOE_F_HOST))

    def shared_router(self, layer, h2, x2, y=True, logits=True, stream=None, sync=False):
        """(y bf16 [T,H] = bf16(x2 + shared(h2)), logits f32 [T,E] = h2 . Wr^T) on the device
        (dense/shared.rs:1-3); either may be skipped."""
        h = as_bf16(h2)
        T = h.shape[0]
        x = as_bf16(x2) if y else None
        yo = torch.empty(T, self.H, dtype=torch.bfloat16, device=h.device) if y else None
        lo = torch.empty(T, self.E, dtype=torch.float32, device=h.device) if logits else None
        check(lib().moe_shared_router(self._h, layer, T, _vp(h), _vp(x), _vp(yo), _vp(lo), MOE_F_SYNC if sync else 0,
                                      _stream_ptr(stream, h.device)))
        return yo, lo

    def combine_residual(self, y, moe_out, extra=None, stream=None, sync=False):
        """x_next bf16 [T,H] = bf16((y + extra) + moe_out) (dense/combine.rs:1)."""
        yy = as_bf16(y)
        m = _as(moe_out, torch.float32)
        e = None if extra is None else _as(extra, torch.float32)
        T = yy.shape[0]
        xn = torch.empty(T, self.H, dtype=torch.bfloat16, device=yy.device)
        check(lib().moe_combine_residual(self._h, T, _vp(yy), _vp(e), _vp(m), _vp(xn), MOE_F_SYNC if sync else 0,
                                         _stream_ptr(stream, yy.device)))
        return xn

    def block_forward(self, layer, h2, x2, extra=None, return_parts=False, stream=None, sync=False):
        """One MoE block: x_next = bf16((bf16(x2 + shared(h2)) + extra) + routed(h2, h2 . Wr^T)).
        Device tensors in, device x_next out (with y and the logits when return_parts)."""
        h = as_bf16(h2)
        x = as_bf16(x2)
        e = None if extra is None else _as(extra, torch.float32)
        T = h.shape[0]
        xn = torch.empty(T, self.H, dtype=torch.bfloat16, device=h.device)
        yo = torch.empty(T, self.H, dtype=torch.bfloat16, device=h.device) if return_parts else None
        lo = torch.empty(T, self.E, dtype=torch.float32, device=h.device) if return_parts else None
        check(lib().moe_block_forward(self._h, layer, T, _vp(h), _vp(x), _vp(e), _vp(xn), _vp(yo), _vp(lo),
                                      MOE_F_SYNC if sync else 0, _stream_ptr(stream, h.device)))
        return (xn, yo, lo) if return_parts else xn

    def block_forward_host(self, layer, h2, x2, extra=None):
        """block_forward with host buffers (synchronous): returns x_next as a CPU bf16 tensor."""
        h = as_bf16(h2).cpu()
        x = as_bf16(x2).cpu()
        e = None if extra is None else _as(extra, torch.float32).cpu()
        xn = torch.empty(h.shape[0], self.H, dtype=torch.bfloat16)
        check(lib().moe_block_forward(self._h, layer, h.shape[0], _vp(h), _vp(x), _vp(e), _vp(xn), None, None,
                                      MOE_F_HOST, _stream_ptr(None, self.device)))
        return xn

    def forward_host(self, layer, hidden, logits, out=None, return_topk=False, accumulate=False):
        """Host buffers in and out (numpy or CPU tensors).  On the fused path pinned logits and
        16-byte-aligned pinned outputs are used in place by the kernels; others are staged."""
        x = as_bf16(hidden)
        lg = _as(logits, torch.float32)
        T = x.shape[0]
        if out is None:
            out = torch.empty(T, self.H, dtype=torch.float32)
        idx = w = None
        if return_topk:
            idx = torch.empty(T, self.K, dtype=torch.int32)
            w = torch.empty(T, self.K, dtype=torch.float32)
        flags = MOE_F_HOST | (MOE_F_ACCUMULATE if accumulate else 0)
        check(lib().moe_forward(self._h, layer, T, _vp(x), _vp(lg), _vp(out), _vp(idx), _vp(w), flags,
                                _stream_ptr(None, self.device)))
        return (out, idx, w) if return_topk else out

    def route(self, logits, bias=None, stream=None):
        """Router + permutation on the GPU; returns a dict of host numpy arrays (synchronous)."""
        lg = _as(logits, torch.float32, self.device)
        T = lg.shape[0]
        b = None if bias is None else self._bias(bias, self.device)
        dev = self.device
        r = dict(idx=torch.empty(T, self.K, dtype=torch.int32, device=dev),
                 w=torch.empty(T, self.K, dtype=torch.float32, device=dev),
                 counts=torch.empty(self.E, dtype=torch.int32, device=dev),
                 offsets=torch.empty(self.E + 1, dtype=torch.int32, device=dev),
                 perm=torch.empty(max(1, T * self.K), dtype=torch.int32, device=dev),
                 job_order=torch.empty(self.E, dtype=torch.int32, device=dev),
                 n_jobs=torch.empty(1, dtype=torch.int32, device=dev))
        status = lib().moe_route(self._h, T, _vp(lg), _vp(b), _vp(r["idx"]), _vp(r["w"]), _vp(r["counts"]),
                                 _vp(r["offsets"]), _vp(r["perm"]), _vp(r["job_order"]), _vp(r["n_jobs"]), MOE_F_SYNC,
                                 _stream_ptr(stream, dev))
        res = {k: v.cpu().numpy() for k, v in r.items()}
        res["perm"] = res["perm"][:T * self.K]
        res["job_order"] = res["job_order"][:int(res["n_jobs"][0])]
        res["status"] = status
        return res

    # ---- reference CPU-kernel surfaces ----
    def experts(self, x, gus, ds, toks, ws, out=None, accumulate=False, stream=None):
        """cpu_moe surface with device-resident weights: out[T,H] fp32 (device)."""
        xd = as_bf16(x, self.device)
        T = xd.shape[0]
        gus = [as_bf16(g, self.device) for g in gus]
        ds = [as_bf16(d, self.device) for d in ds]
        n = len(gus)
        off = np.zeros(n + 1, np.int64)
        for j, t in enumerate(toks):
            off[j + 1] = off[j] + len(t)
        tk = np.ascontiguousarray(np.concatenate([np.asarray(_cpu(t), np.int64) for t in toks]) if n else np.zeros(1, np.int64))
        wv = np.ascontiguousarray(np.concatenate([np.asarray(_cpu(w), np.float32) for w in ws]) if n else np.zeros(1, np.float32))
        gp = (ctypes.c_void_p * max(1, n))(*[g.data_ptr() for g in gus])
        dp = (ctypes.c_void_p * max(1, n))(*[d.data_ptr() for d in ds])
        if out is None:
            out = torch.empty(T, self.H, dtype=torch.float32, device=self.device)
        flags = MOE_F_ACCUMULATE if accumulate else 0
        check(lib().moe_experts(self._h, T, _vp(xd), n, gp, dp, off.ctypes.data_as(ctypes.c_void_p),
                                tk.ctypes.data_as(ctypes.c_void_p), wv.ctypes.data_as(ctypes.c_void_p), _vp(out),
                                flags, _stream_ptr(stream, self.device)))
        self._keep = (gus, ds)
        return out

    def ck_moe3(self, bases, w, x, out, stream=None):
        """ck_moe3: out[H] += sum_e w[e] * expert_e(x); bases = device bf16 tensors [3*F*H]."""
        n = len(bases)
        bp = (ctypes.c_void_p * max(1, n))(*[b.data_ptr() for b in bases])
        wd = _as(w, torch.float32, self.device)
        xd = as_bf16(x, self.device)
        check(lib().moe_ck_moe3(self._h, n, bp, _vp(wd), _vp(xd), _vp(out), 0, _stream_ptr(stream, self.device)))
        return out

    def ck_moe_q8w(self, qs, scs, w, x, out, stream=None):
        n = len(qs)
        qp = (ctypes.c_void_p * max(1, n))(*[q.data_ptr() for q in qs])
        sp = (ctypes.c_void_p * max(1, n))(*[s.data_ptr() for s in scs])
        wd = _as(w, torch.float32, self.device)
        xd = as_bf16(x, self.device)
        check(lib().moe_ck_moe_q8w(self._h, n, qp, sp, _vp(wd), _vp(xd), _vp(out), 0, _stream_ptr(stream, self.device)))
        return out

    def place_expert_q8(self, g, u, d, stream=None):
        """ck_place_expert_q8 on the GPU -> (q int8 [3FH], sc fp32 [2F+H], rs int32 [2F+H]) device tensors."""
        g, u, d = (as_bf16(a, self.device) for a in (g, u, d))
        q = torch.empty(3 * self.F * self.H, dtype=torch.int8, device=self.device)
        sc = torch.empty(2 * self.F + self.H, dtype=torch.float32, device=self.device)
        rs = torch.empty(2 * self.F + self.H, dtype=torch.int32, device=self.device)
        check(lib().moe_place_expert_q8(self._h, _vp(g), _vp(u), _vp(d), _vp(q), _vp(sc), _vp(rs), MOE_F_SYNC,
                                        _stream_ptr(stream, self.device)))
        return q, sc, rs

    # ---- 8-bit floating point: e4m3 values with one scale for each 128 ----
    # Checks, allocation and the C calls of these methods (but route_topk) are in _torch_binding: at one token the GPU
    # takes a few microseconds, and Python with ctypes took longer than that.
    def quantize_fp8(self, x, block_rows=1, stream=None):
        """x [..., rows, cols] bf16 or fp32 -> Fp8(q, scale): one scale for each 128 columns of a row
        (block_rows=1, activations) or of 128 rows (block_rows=128, weights).  Scales are powers of two;
        infinities and NaN become NaN.  cols must be a multiple of 16."""
        if stream is not None:
            with self._on(stream):
                return self.quantize_fp8(x, block_rows)
        p = self._plane or self._bind()
        return Fp8(*_calls.quantize_fp8(p, _tensor("x", x), block_rows, _raw_stream(self._index)))

    def matmul_fp8(self, x, w, out_dtype=torch.bfloat16, out=None, stream=None):
        """out [M, N] = x [M, K] . w [N, K]^T with fp32 sums.  x: Fp8 with a scale per row and 128 columns
        (or a bf16 / fp32 tensor, which is quantised first); w: Fp8 with a scale per 128 x 128 block."""
        if stream is not None:
            with self._on(stream):
                return self.matmul_fp8(x, w, out_dtype, out)
        if type(x) is not Fp8:
            x = self.quantize_fp8(x)
        p = self._plane or self._bind()
        return _calls.matmul_fp8(p, x.q, x.scale, *_fp8("w", w), out_dtype, out, _raw_stream(self._index))

    def experts_fp8(self, x, gate_up, down, idx, w, out_dtype=torch.float32, out=None, accumulate=False, stream=None):
        """The routed experts on e4m3 weights: out [T, H] = sum_k w[t, k] expert_idx[t, k](x[t]).

        x [T, H] bf16; gate_up Fp8 [E, 2, F, H] (gate rows, up rows) and down Fp8 [E, H, F], scales per
        128 x 128 block; idx [T, top_k] int32 (negative: no expert) and w [T, top_k] fp32, as
        route_topk() gives them.  Tokens and SwiGLU activations are quantised per row and 128 columns."""
        if stream is not None:
            with self._on(stream):
                return self.experts_fp8(x, gate_up, down, idx, w, out_dtype, out, accumulate)
        p = self._plane or self._bind()
        return _calls.experts_fp8(p, x, *_fp8("gate_up", gate_up), *_fp8("down", down), idx, w, out_dtype, out, accumulate,
                                  _raw_stream(self._index))

    def route_topk(self, logits, bias=None, stream=None):
        """The router alone, on the device and without a wait: (idx [T, top_k] int32, w [T, top_k] fp32).

        Written straight into the results: calls on several streams or in captured graphs may overlap, and T
        is not bound by max_tokens."""
        if stream is not None:
            with self._on(stream):
                return self.route_topk(logits, bias)
        if isinstance(logits, torch.Tensor) and logits.requires_grad and torch.is_grad_enabled():
            raise ValueError("route_topk records no autograd graph: pass logits.detach(), or call under torch.no_grad()")
        lg = _as(logits, torch.float32, self.device)
        if lg.dim() != 2 or lg.shape[1] != self.E:
            raise ValueError(f"logits are {tuple(lg.shape)}, the context has {self.E} experts")
        T = lg.shape[0]
        b = None if bias is None else self._bias(bias, self.device)
        idx = torch.empty(T, self.K, dtype=torch.int32, device=self.device)
        w = torch.empty(T, self.K, dtype=torch.float32, device=self.device)
        check(lib().moe_route_topk(self._h, T, _vp(lg), _vp(b), _vp(idx), _vp(w), 0, _raw_stream(self._index)))
        return idx, w

    def route_groups(self, logits, groups, top_groups, bias=None, renormalize=True, scale=1.0, stream=None):
        """The router limited to the best groups of experts: (idx [T, top_k] int32, w [T, top_k] fp32), on the device.

        logits [T, E] fp32; `groups` groups of E / groups neighbours, of which the top_groups best are open: by their largest
        logit (softmax scoring), or by the sum of their two largest s + bias (sigmoid; bias [E] fp32 only selects).  Then the
        top_k best experts of those, the best first, ties to the lower index; w = scale * softmax probability or s, divided by
        the chosen ones' sum where renormalize is set.  A logit of -inf masks under softmax; under sigmoid a bias of -inf, or one well below
        the others (faster), does.  The weights' gradient is route_backward()."""
        if stream is not None:
            with self._on(stream):
                return self.route_groups(logits, groups, top_groups, bias, renormalize, scale)
        p = self._plane or self._bind()
        return _calls.route_groups(p, _tensor("logits", logits), groups, top_groups, bias, renormalize, scale, _raw_stream(self._index))

    def route_backward(self, logits, idx, dw, renormalize=True, scale=1.0, out=None, accumulate=False, stream=None):
        """dlogits [T, E] fp32 from dw [T, top_k], the gradient of route_groups()'s or route_topk()'s weights at idx (negative:
        no choice); renormalize and scale as they were routed with.  accumulate: out +=, as behind balance_loss_backward()."""
        if stream is not None:
            with self._on(stream):
                return self.route_backward(logits, idx, dw, renormalize, scale, out, accumulate)
        p = self._plane or self._bind()
        return _calls.route_backward(p, _tensor("logits", logits), _tensor("idx", idx), _tensor("dw", dw), renormalize, scale, out, accumulate,
                                     _raw_stream(self._index))

    # ---- the router's load-balance loss ----
    def balance_loss(self, logits, idx, offsets=None, mask=None, stream=None):
        """(loss, BalanceStats): the router's load-balance loss over each sequence, and per-expert counts.

        logits [T, E] fp32, idx [T, top_k] int32 choices (negative: none); offsets [B + 1] int32: the
        sequences' first tokens (None: one sequence); mask [T] bool: tokens that count (None: all).
        loss = mean over sequences of sum_e f_e P_e, f_e = E * share of the choices, P_e = mean score.
        No autograd graph is recorded: the gradient is balance_loss_backward()."""
        if stream is not None:
            with self._on(stream):
                return self.balance_loss(logits, idx, offsets, mask)
        p = self._plane or self._bind()
        loss, *stats = _calls.balance_loss(p, logits, idx, offsets, mask, _raw_stream(self._index))
        return loss, BalanceStats(*stats)

    def balance_loss_backward(self, logits, stats, grad=None, out=None, stream=None):
        """dlogits [T, E] fp32 = grad * d loss / d logits (grad: a device fp32 scalar; None: 1), zero for
        tokens that do not count.  logits and stats are those of balance_loss()."""
        if stream is not None:
            with self._on(stream):
                return self.balance_loss_backward(logits, stats, grad, out)
        p = self._plane or self._bind()
        return _calls.balance_loss_backward(p, logits, *stats, grad, out, _raw_stream(self._index))

    # ---- residual addition and root-mean-square norm ----
    def add_norm(self, x, weight, residual=None, eps=1e-6, out_dtype=torch.bfloat16, fp8=False, stream=None):
        """Normed(y, fp8, sum, rstd): sum = x + residual in the residual's type, y = sum / sqrt(mean sum^2 + eps) * weight.

        x, residual [..., C] and weight [C] bf16 or fp32; C at most 16384.  out_dtype: bf16, fp32, or None for no y;
        fp8: y also as e4m3 with a scale for each 128 columns (C a multiple of 16), as matmul_fp8 takes it, rounded
        from y before that is.  No autograd graph is recorded: the gradient is add_norm_backward()."""
        if stream is not None:
            with self._on(stream):
                return self.add_norm(x, weight, residual, eps, out_dtype, fp8)
        p = self._plane or self._bind()
        y, q, scale, total, rstd = _calls.add_norm(p, _tensor("x", x), _tensor("weight", weight), residual, eps, out_dtype, fp8,
                                                   _raw_stream(self._index))
        return Normed(y, None if q is None else Fp8(q, scale), total, rstd)

    def add_norm_backward(self, dy, sum, weight, rstd, dsum=None, weight_grad=True, stream=None):
        """(dx, dweight) of add_norm: dy [..., C] (bf16 or fp32) is the gradient of y, dsum (sum's type) what else flows into
        the sum; dx, of sum's type, is the gradient of x and of the residual; dweight [C] fp32 (weight_grad=False: None)."""
        if stream is not None:
            with self._on(stream):
                return self.add_norm_backward(dy, sum, weight, rstd, dsum, weight_grad)
        p = self._plane or self._bind()
        return _calls.add_norm_backward(p, _tensor("dy", dy), _tensor("sum", sum), _tensor("weight", weight), _tensor("rstd", rstd), dsum,
                                        weight_grad, _raw_stream(self._index))

    # ---- low-rank adapters beside a shared projection ----
    def add_lora(self, base, x, a, b, ids, scale=None, out=None, stream=None):
        """out [T, N] = base + scale[i] * (x . a[i]^T) . b[i]^T for each token's adapter i = ids[t] (negative: base alone).

        base [T, N] (bf16 or fp32) is the shared projection of x [T, K] bf16, matmul_fp8()'s result for instance; a [n, r, K]
        and b [n, N, r] bf16, contiguous; K and r multiples of 8, r at most 128; ids [T] int32; scale [n] fp32 (None: 1).
        fp32 sums, rounded at the end; for bf16 results calls of many tokens (more than 128 up to r = 32, 64 up to r = 64, 32 beyond)
        hold scale[i] * (x . a[i]^T) to 2^-16.  out may be base: tokens without an adapter are then left as they are."""
        if stream is not None:
            with self._on(stream):
                return self.add_lora(base, x, a, b, ids, scale, out)
        p = self._plane or self._bind()
        return _calls.add_lora(p, _tensor("base", base), _tensor("x", x), _tensor("a", a), _tensor("b", b), _tensor("ids", ids), scale, out,
                               _raw_stream(self._index))

    def _on(self, stream):
        if stream.device != self.device:
            raise ValueError(f"stream is on {stream.device}, the context on {self.device}")
        return torch.cuda.stream(stream)

    def _bind(self):
        """What the calls of _torch_binding need of this context; dropped with it by close()."""
        global _calls
        if _calls is None:
            lib()  # the library first: the binding is linked to it
            _calls = _load_binding()
        self._plane = _calls.Plane(self._h.value if self._h else 0, self.device, self.H, self.F, self.E, self.K)
        return self._plane

    def status(self, stream=None):
        return lib().moe_status(self._h, _stream_ptr(stream, self.device))

    @property
    def launch_count(self):
        return int(lib().moe_launch_count(self._h))

    def set_option(self, option, value):
        check(lib().moe_set_option(self._h, int(option), int(value)))

    def timeline(self):
        """Per-CTA phase stamps of the latest fused launch (MOE_OPT_TIMELINE on): [SMs, 24] ns."""
        sms = torch.cuda.get_device_properties(self.device).multi_processor_count
        n = sms * 24 + 3 * 1024
        buf = np.zeros(n, np.uint64)
        check(lib().moe_timeline_read(self._h, buf.ctypes.data_as(ctypes.c_void_p), n))
        self.stage_log = buf[sms * 24:].reshape(3, 1024)
        return buf[:sms * 24].reshape(-1, 24)

    def profile(self, enable=True):
        check(lib().moe_profile(self._h, int(bool(enable))))

    def profile_read(self, n_stages=4):
        """Summed ms per stage (route, gate/up, down, combine) of the profiled forwards, and their count."""
        ms = (ctypes.c_double * n_stages)()
        n = ctypes.c_int64()
        check(lib().moe_profile_read(self._h, ms, n_stages, ctypes.byref(n)))
        return list(ms), int(n.value)


def _load_binding():
    path = binding_path()
    if not os.path.exists(path):
        raise ImportError(f"{path} is missing: build it with `python -m npu_offload_b200.build` for this Python and torch")
    spec = importlib.util.spec_from_file_location(__package__ + "._torch_binding", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def _tensor(name, t):
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{name} must be a tensor on the GPU, not {type(t).__name__}")
    return t


def _fp8(name, m):
    if type(m) is not Fp8:
        raise ValueError(f"{name} must be an Fp8, as quantize_fp8 gives it")
    return m


def _cpu(t):
    return t.cpu() if isinstance(t, torch.Tensor) else t


# ---------------- cpu_moe_ext drop-in ----------------
_planes = {}


class _WeightCache:
    """Device copies of CPU weight tensors for gpu_moe, keyed on the tensor object itself.

    An entry holds a weak reference to the host tensor and the tensor's version counter
    (``Tensor._version``, bumped by every in-place write), so a tensor that is freed (its storage
    possibly reused at the same address) or overwritten in place (the reference's expert swap,
    runtime.py:287-311) is copied again instead of returning stale weights.  Entries die with their
    host tensor, and the cache keeps at most ``limit_bytes`` of device copies, evicting the least
    recently used first.
    """

    def __init__(self, limit_bytes):
        import collections
        self.limit = int(limit_bytes)
        self.bytes = 0
        self.entries = collections.OrderedDict()  # id(t) -> (weakref, version, device, copy)

    def _drop(self, key):
        e = self.entries.pop(key, None)
        if e is not None:
            self.bytes -= e[3].numel() * e[3].element_size()

    def get(self, t, device):
        import weakref
        key = id(t)
        e = self.entries.get(key)
        if e is not None and e[0]() is t and e[1] == t._version and e[2] == device:
            self.entries.move_to_end(key)
            return e[3]
        self._drop(key)
        d = as_bf16(t, device)
        nb = d.numel() * d.element_size()
        while self.entries and self.bytes + nb > self.limit:
            self._drop(next(iter(self.entries)))
        if nb <= self.limit:
            ref = weakref.ref(t, lambda _r, k=key, c=self: c._drop(k) if k in c.entries and c.entries[k][0] is _r else None)
            self.entries[key] = (ref, t._version, device, d)
            self.bytes += nb
        return d

    def clear(self):
        self.entries.clear()
        self.bytes = 0


# device copies of CPU weights: 8 GiB by default (NPU_OFFLOAD_GPU_MOE_CACHE_GB overrides)
_wcache = _WeightCache(float(__import__("os").environ.get("NPU_OFFLOAD_GPU_MOE_CACHE_GB", "8")) * (1 << 30))


def _plane_for(device, H, F, pairs, T, n_jobs):
    key = (device.index, H, F)
    p = _planes.get(key)
    if p is None or p.max_tokens * p.K < pairs or p.max_tokens < T or p.E < n_jobs:
        if p is not None:
            p.close()
        mt = 64
        while mt * 16 < pairs or mt < T:
            mt *= 2
        # scratch capacity is max_tokens * top_k pairs (top_k=16 needs n_experts >= 16)
        ne = 16
        while ne < n_jobs:
            ne *= 2
        if ne > 256:
            raise RuntimeError("gpu_moe supports at most 256 experts per call")
        p = MoEDataPlane(H, F, n_experts=ne, top_k=16, n_layers=1, max_tokens=min(mt, 4096), device=device)
        _planes[key] = p
    return p


def _device_weight(t, device):
    if t.is_cuda:
        return as_bf16(t)
    return _wcache.get(t, device)


def gpu_moe(x, gus, ds, toks, ws):
    """Drop-in for ``cpu_moe_ext.ext.cpu_moe`` (solar_hybrid/cpu_moe.cpp:38-96).

    x [T,H] bf16; gus[e] [2F,H] bf16 (gate rows then up rows); ds[e] [H,F] bf16; toks[e] int64 token
    rows; ws[e] fp32 routing weights.  Returns out [T,H] fp32 = sum_e ws[e] * expert_e(x[toks[e]]),
    on x's device (a CPU x gives a CPU result, as the reference does).  CPU weight tensors are copied
    to the GPU and cached per tensor object and version (a bounded cache: see _WeightCache); pass
    CUDA tensors to avoid the cache.
    """
    T, H = x.shape
    E = len(gus)
    if E == 0:
        return torch.zeros(T, H, dtype=torch.float32, device=x.device)
    F = ds[0].shape[1]
    if H % 32 != 0 or F % 32 != 0:
        raise RuntimeError("H,F must be multiples of 32")
    if H % 256 != 0 or F % 64 != 0:
        raise RuntimeError("gpu_moe needs H % 256 == 0 and F % 64 == 0")
    device = x.device if x.is_cuda else torch.device("cuda", torch.cuda.current_device())
    pairs = sum(len(t) for t in toks)
    plane = _plane_for(device, H, F, pairs, T, E)
    g = [_device_weight(a, device) for a in gus]
    d = [_device_weight(a, device) for a in ds]
    out = plane.experts(x, g, d, toks, ws)
    return out if x.is_cuda else out.cpu()


def set_threads(n):
    """Accepted for compatibility with cpu_moe_ext.set_threads; the GPU path has no host thread pool."""
    return None
