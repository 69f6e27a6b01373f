"""torch.autograd bindings of the HIP kernels (host-side plumbing only: pointers, streams, saved tensors).

Every function here requires CUDA(HIP) float32 tensors and calls libmbvae_hip.so through ctypes; nothing
falls back to eager PyTorch arithmetic.
"""
import math
import os

import torch

from . import _lib

MASK_NONE, MASK_NODE, MASK_EDGE = 0, 1, 2
# A/B aid: below the edge-tensor shapes, add a residual gradient in a separate pass instead of the tiled product's epilogue
_NO_GENERIC_ADDEND = os.environ.get("MBVAE_NO_GENERIC_ADDEND", "0") not in ("", "0")

# Opt-in reduced-precision STORAGE of the training step's largest activations (the edge block's [bs,n,n,2dx]
# projection output and its gradient, the attention output P [bs,n,n,dx] and its gradient): bf16 in memory, fp32
# weights, fp32 arithmetic and accumulation everywhere.  Off by default: the default path is fp32 end to end.
_BF16_STORAGE = os.environ.get("MBVAE_BF16_STORAGE", "0") not in ("", "0")


def set_bf16_storage(on):
    """Switch the bf16 storage mode of the edge block on or off (takes effect at the next forward)."""
    global _BF16_STORAGE
    _BF16_STORAGE = bool(on)


def bf16_storage():
    return _BF16_STORAGE


# Opt-in: the feature encoders and the drug / target fusion run each gate or residual update together with the LayerNorm that
# opens the next block (gated_residual_norm) instead of as separate kernels.  Same function and the same dropout masks; sums in another
# order, so results agree to fp32 rounding and not bit for bit.
_FUSED_BLOCKS = os.environ.get("MBVAE_FUSED_BLOCKS", "0") not in ("", "0")


def set_fused_blocks(on):
    """Switch the fused block updates of the encoders and the fusion on or off (takes effect at the next forward)."""
    global _FUSED_BLOCKS
    _FUSED_BLOCKS = bool(on)


def fused_blocks():
    return _FUSED_BLOCKS

_ws_cache = {}


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def workspace(device, nbytes=160 << 20):
    """Scratch buffer per (device, stream), shared by all kernels issued on that stream (which serialises them)."""
    key = (device.index if device.index is not None else torch.cuda.current_device(), _stream())
    ws = _ws_cache.get(key)
    if ws is None or ws.numel() < nbytes:
        ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
        _ws_cache[key] = ws
    return ws


_queue_cache = {}


def _work_counter(device):
    """One int32 per device for kernels that hand out their tasks through a counter (they run serialised on the stream
    and zero it themselves)."""
    key = (device.index if device.index is not None else torch.cuda.current_device(), _stream())
    q = _queue_cache.get(key)
    if q is None:
        q = _queue_cache[key] = torch.zeros(1, dtype=torch.int32, device=device)
    return q


_side_streams = {}
_SIDE_STREAM = [os.environ.get("MBVAE_SIDE_STREAM", "0") not in ("", "0")]      # (the test suite runs both ways)


if _SIDE_STREAM[0] and hasattr(torch.autograd.graph, "set_warn_on_accumulate_grad_stream_mismatch"):
    torch.autograd.graph.set_warn_on_accumulate_grad_stream_mismatch(False)      # (intended, see set_side_stream)


def set_side_stream(on):
    """Training: run the node / global-feature remainder of a transformer layer (small, latency-bound kernels) on a
    second HIP stream next to the layer's long edge-tensor kernels.  Same kernels, same sums: results are bit-identical
    to one stream.  Not used while a HIP graph is being captured; gradient-sync hooks order their collectives behind
    both streams (ddp.BucketedGradSync)."""
    _SIDE_STREAM[0] = bool(on)
    if on and hasattr(torch.autograd.graph, "set_warn_on_accumulate_grad_stream_mismatch"):
        # parameter gradients produced on the second stream are accumulated on the parameters' own stream: intended
        torch.autograd.graph.set_warn_on_accumulate_grad_stream_mismatch(False)


def side_stream(device):
    """The device's second stream when set_side_stream(True) and nothing is being captured, else None."""
    if not _SIDE_STREAM[0] or torch.cuda.is_current_stream_capturing():
        return None
    key = device.index if device.index is not None else torch.cuda.current_device()
    st = _side_streams.get(key)
    if st is None:
        st = _side_streams[key] = torch.cuda.Stream(device=device)      # (a high-priority stream measured the same)
    return st


def option_set(name):
    """Current value of a process-wide library switch (mbvae_get_option) as a bool."""
    return _lib.load().mbvae_get_option(name.encode()) > 0


def _f32c(t, name="tensor"):
    if not t.is_cuda or t.dtype != torch.float32:
        raise RuntimeError(f"{name}: expected a float32 tensor on the GPU (got {t.dtype} on {t.device}); "
                           "the HIP path has no CPU fallback")
    return t if t.is_contiguous() else t.contiguous()


def _mask_u8(mask):
    if mask is None:
        return None
    m = mask if mask.is_contiguous() else mask.contiguous()
    return m.view(torch.uint8) if m.dtype == torch.bool else m.to(torch.uint8)


# ------------------------------------------------------------------------------------------------ linear
class _Linear(torch.autograd.Function):
    """with_alias: also returns an alias of x for a second consumer (a residual branch); the alias' gradient is then
    folded into the input-gradient product's epilogue instead of meeting it in a separate accumulation pass."""

    @staticmethod
    def forward(ctx, x, w, b, act, mask, mask_mode, n_nodes, drop_p, seed, with_alias, in_gate_scale, pregated):
        """in_gate_scale (float or None): x came out of ReLU (+ dropout with that keep scale) of the layer below and has
        no other consumer: this layer's backward applies that gate to the input gradient it produces.  pregated: the
        counterpart on the layer below (act == 1): its dy arrives already gated."""
        bf16_in = x.dtype == torch.bfloat16          # bf16 storage mode: the attention output P feeding e_out
        if bf16_in:
            if not x.is_cuda or act or drop_p > 0 or with_alias:
                raise RuntimeError("a bf16 input is only supported for a plain Linear on the GPU (the e_out projection)")
            x2 = x.contiguous().reshape(-1, x.shape[-1])
        else:
            x2 = _f32c(x, "x").reshape(-1, x.shape[-1])
        w = _f32c(w, "weight")
        M, K = x2.shape
        N = w.shape[0]
        y = torch.empty((M, N), dtype=torch.float32, device=x.device)
        ws = workspace(x.device)
        m8 = _mask_u8(mask)
        if bf16_in:
            _lib.call("mbvae_linear_fwd_bf16", x2.data_ptr(), K, w.data_ptr(), _ptr(b), y.data_ptr(), N, M, K, N,
                      _ptr(m8), mask_mode, n_nodes, _stream(), tag=(M, K, N))
        else:
            _lib.call("mbvae_linear_fwd", x2.data_ptr(), K, w.data_ptr(), _ptr(b), y.data_ptr(), N, M, K, N, act,
                      _ptr(m8), mask_mode, n_nodes, float(drop_p), int(seed), 0, ws.data_ptr(), ws.numel(), _stream(),
                      tag=(M, K, N))
        gated = act == 1 and not pregated
        ctx.save_for_backward(x2, w, y if gated else None, m8)
        ctx.cfg = (mask_mode, n_nodes, float(drop_p), gated, b is not None, x.shape)
        ctx.in_gate_scale = in_gate_scale
        ctx.relu = act == 1
        out = y.reshape(*x.shape[:-1], N)
        return (out, x.view_as(x)) if with_alias else out

    @staticmethod
    def backward(ctx, dy, dres=None):
        x2, w, gate, m8 = ctx.saved_tensors
        mask_mode, n_nodes, drop_p, gated, has_bias, xshape = ctx.cfg
        M, K = x2.shape
        N = w.shape[0]
        dy2 = _f32c(dy, "dy").reshape(M, N)
        ws = workspace(dy.device)
        gscale = 1.0 / (1.0 - drop_p) if (gated and drop_p > 0) else 1.0
        # a ReLU gate (y > 0) already implies the row mask (also when the layer above has applied it to dy)
        mm = MASK_NONE if ctx.relu else mask_mode
        dx = dw = db = None
        if x2.dtype == torch.bfloat16:               # bf16 storage mode: dx leaves as bf16, x is read as bf16
            if ctx.needs_input_grad[0]:
                dx = torch.empty((M, K), dtype=torch.bfloat16, device=dy.device)
                _lib.call("mbvae_linear_bwd_input_bf16", dy2.data_ptr(), 0, N, w.data_ptr(), 0, dx.data_ptr(), 1, K, M, K, N,
                          _ptr(m8), mm, n_nodes, _stream(), tag=(M, K, N))
                dx = dx.reshape(xshape)
            need_db = has_bias and ctx.needs_input_grad[2]
            if ctx.needs_input_grad[1] or need_db:
                dw = torch.empty((N, K), dtype=torch.float32, device=dy.device)
                db = torch.empty((N,), dtype=torch.float32, device=dy.device) if need_db else None
                _lib.call("mbvae_linear_bwd_weight_bf16", dy2.data_ptr(), 0, N, x2.data_ptr(), 1, K, dw.data_ptr(), _ptr(db),
                          M, K, N, _ptr(m8), mm, n_nodes, ws.data_ptr(), ws.numel(), _stream(), tag=(M, K, N))
                if not ctx.needs_input_grad[1]:
                    dw = None
            return dx, dw, db, None, None, None, None, None, None, None, None, None
        if ctx.needs_input_grad[0] and ctx.in_gate_scale is not None:
            dx = torch.empty((M, K), dtype=torch.float32, device=dy.device)
            _lib.call("mbvae_linear_bwd_input_outgate", dy2.data_ptr(), N, w.data_ptr(), dx.data_ptr(), K, M, K, N, x2.data_ptr(),
                      float(ctx.in_gate_scale), _ptr(m8), mm, n_nodes, ws.data_ptr(), ws.numel(), _stream(), tag=(M, K, N))
            if dres is not None:
                dx += _f32c(dres, "dres").reshape(M, K)
            dx = dx.reshape(xshape)
        elif ctx.needs_input_grad[0]:
            dx = torch.empty((M, K), dtype=torch.float32, device=dy.device)
            folded = False
            if dres is not None:
                dres = _f32c(dres, "dres").reshape(M, K)
            if dres is not None and (M >= 32768 or not _NO_GENERIC_ADDEND):
                folded = _lib.call("mbvae_linear_bwd_input_add", dy2.data_ptr(), N, w.data_ptr(), dres.data_ptr(), dx.data_ptr(), K,
                                   M, K, N, _ptr(gate), gscale, _ptr(m8), mm, n_nodes, _stream(), tag=(M, K, N),
                                   allow_unsupported=True)
            if not folded:
                _lib.call("mbvae_linear_bwd_input", dy2.data_ptr(), N, w.data_ptr(), dx.data_ptr(), K, M, K, N, _ptr(gate),
                          gscale, _ptr(m8), mm, n_nodes, 0, ws.data_ptr(), ws.numel(), _stream(), tag=(M, K, N))
                if dres is not None:
                    dx += dres
            dx = dx.reshape(xshape)
        need_db = has_bias and ctx.needs_input_grad[2]
        if ctx.needs_input_grad[1] or need_db:     # (a frozen weight with a trainable bias still needs the column sums)
            dw = torch.empty((N, K), dtype=torch.float32, device=dy.device)
            db = torch.empty((N,), dtype=torch.float32, device=dy.device) if need_db else None
            _lib.call("mbvae_linear_bwd_weight", dy2.data_ptr(), N, x2.data_ptr(), K, dw.data_ptr(), _ptr(db), M, K, N,
                      _ptr(gate), gscale, _ptr(m8), mm, n_nodes, 0, ws.data_ptr(), ws.numel(), _stream(), tag=(M, K, N))
            if not ctx.needs_input_grad[1]:
                dw = None
        return dx, dw, db, None, None, None, None, None, None, None, None, None


def linear(x, weight, bias=None, act=0, mask=None, mask_mode=MASK_NONE, n_nodes=0, drop_p=0.0, seed=0, with_alias=False,
           in_gate_scale=None, pregated=False):
    """y = rowmask(dropout(act(x @ W^T + b))); act: 0 none, 1 ReLU.  Dropout is only supported after ReLU.
    with_alias=True returns (y, alias of x): use the alias for x's other consumer (residual branch).
    in_gate_scale / pregated: see ffn() - a ReLU layer's gate applied by the backward of its only consumer."""
    if drop_p > 0 and act != 1:
        raise ValueError("dropout in the GEMM epilogue is only implemented after ReLU")
    if mask is None:
        mask_mode = MASK_NONE
    if pregated and act != 1:
        raise ValueError("pregated is the counterpart of a ReLU layer")
    return _Linear.apply(x, weight, bias, act, mask, mask_mode, n_nodes, drop_p, seed, with_alias, in_gate_scale, pregated)


class _FfnLn(torch.autograd.Function):
    """LayerNorm(x + dropout(l2(dropout(relu(l1(x)))))) of the edge tensor in ONE forward kernel
    (mbvae_edge_ffn_fwd_train): the hidden activation and the pre-LayerNorm sum are written once for the backward and
    never read back in the forward.  The backward is the one of _Linear (l1, gate handed over) followed by _LinearLn
    (l2), run from here on the stored tensors: same kernels, same dropout masks."""

    class _LinCtx:                       # what _Linear.backward reads from its ctx
        pass

    @staticmethod
    def forward(ctx, x, w1, b1, w2, b2, gamma, beta, eps, p1, seed1, p2, seed2):
        x2 = _f32c(x, "x").reshape(-1, x.shape[-1])
        w1, w2, gamma, beta = _f32c(w1, "weight"), _f32c(w2, "weight"), _f32c(gamma), _f32c(beta)
        M, d = x2.shape
        dff = w1.shape[0]
        h = torch.empty((M, dff), dtype=torch.float32, device=x.device)
        z, y = torch.empty_like(x2), torch.empty_like(x2)
        _lib.call("mbvae_edge_ffn_fwd_train", x2.data_ptr(), w1.data_ptr(), _ptr(b1), w2.data_ptr(), _ptr(b2), gamma.data_ptr(),
                  beta.data_ptr(), h.data_ptr(), z.data_ptr(), y.data_ptr(), M, d, dff, float(eps), float(p1), int(seed1),
                  float(p2), int(seed2), _stream(), tag=(M, d, dff))
        ctx.save_for_backward(x2, w1, w2, h, z, gamma)
        ctx.cfg = (float(eps), float(p1), float(p2), int(seed2), b1 is not None, b2 is not None, x.shape)
        return y.reshape(x.shape)

    @staticmethod
    def backward(ctx, dy):
        x2, w1, w2, h, z, gamma = ctx.saved_tensors
        eps, p1, p2, seed2, has_b1, has_b2, xshape = ctx.cfg
        rows, D = z.shape
        dy = _f32c(dy, "dy")
        dres = torch.empty_like(z)
        dr = torch.empty_like(z) if p2 > 0 else None
        dgamma, dbeta = torch.empty_like(gamma), torch.empty_like(gamma)
        ws = workspace(z.device)
        _lib.call("mbvae_ln_sum_bwd", z.data_ptr(), gamma.data_ptr(), dy.data_ptr(), dres.data_ptr(), _ptr(dr),
                  dgamma.data_ptr(), dbeta.data_ptr(), rows, D, eps, p2, seed2, ws.data_ptr(), ws.numel(), _stream())
        need = ctx.needs_input_grad
        gscale = 1.0 / (1.0 - p1) if p1 > 0 else 1.0
        dlin = dr if dr is not None else dres
        # activations' gradients in one pass: dh (l1's ReLU / dropout gate applied, h itself is the gate) and dx
        dh = torch.empty_like(h)
        dx = torch.empty_like(x2)
        fused = _lib.call("mbvae_edge_ffn_bwd_data", dlin.data_ptr(), dres.data_ptr(), h.data_ptr(), w1.data_ptr(), w2.data_ptr(),
                          dh.data_ptr(), dx.data_ptr(), rows, D, h.shape[1], gscale, _stream(), tag=(rows, D, h.shape[1]),
                          allow_unsupported=True)
        lin2 = _FfnLn._LinCtx()          # l2: weight / bias gradients (and dh, gated in the product's epilogue, if not fused)
        lin2.saved_tensors = (h, w2, None, None)
        lin2.cfg = (MASK_NONE, 0, 0.0, False, has_b2, h.shape)
        lin2.in_gate_scale, lin2.relu = gscale, False
        lin2.needs_input_grad = (not fused, need[3], need[4])
        dh2, dw2, db2 = _Linear.backward(lin2, dlin)[:3]
        if not fused:
            dh = dh2
        lin1 = _FfnLn._LinCtx()          # l1: dh arrives gated; unfused, the residual branch's gradient joins in its epilogue
        lin1.saved_tensors = (x2, w1, None, None)
        lin1.cfg = (MASK_NONE, 0, p1, False, has_b1, xshape)
        lin1.in_gate_scale, lin1.relu = None, True
        lin1.needs_input_grad = (need[0] and not fused, need[1], need[2])
        dx1, dw1, db1 = _Linear.backward(lin1, dh, dres)[:3]
        dx = (dx.reshape(xshape) if need[0] else None) if fused else dx1
        return dx, dw1, db1, dw2, db2, dgamma, dbeta, None, None, None, None, None


def ffn_ln_train_supported(x, w1, w2):
    """Shapes mbvae_edge_ffn_fwd_train takes: the edge tensor's feed-forward block (64 -> 128 -> 64) over >= 32768 rows."""
    M = x.numel() // x.shape[-1]
    return (x.is_cuda and x.dtype == torch.float32 and x.shape[-1] == 64 and tuple(w1.shape) == (128, 64) and tuple(w2.shape) == (64, 128)
            and M >= 32768 and M % 32 == 0 and M * 128 < 0x3fffffff
            and not (option_set("NO_EDGE_FFN_TRAIN") or option_set("NO_FFN_HANDOVER") or option_set("NO_LN_EPILOGUE")
                     or option_set("NO_TSGEMM") or option_set("NO_TSGEMM2")))


def ffn(x, w1, b1, w2, b2, drop_p=0.0, seed=0, handover=None, ln=None):
    """(l2(dropout(relu(l1(x)))), alias of x for the residual branch): the two Linears of a feed-forward block
    (graph_transformer.py:139-146).  The hidden activation h has exactly one consumer, so with `handover` the ReLU /
    dropout gate of l1 is applied by l2's backward where it produces dh (h itself is the gate) and l1's two gradient
    kernels read the gated dh without loading h again: 0.5 KB less traffic per row.  Default: on for the edge path
    (>= 32768 rows), where the gate sits in the product's epilogue; the short node / global paths keep the gate inside
    l1's kernels (one launch fewer).
    ln = (gamma, beta, eps, drop_p, seed) of the residual LayerNorm that follows: where l2 can take it into its epilogue
    (linear_ln_supported) the result is (LayerNorm(x + dropout(l2(.))), None) - the block is finished; the edge tensor's
    block (ffn_ln_train_supported) runs as one forward kernel."""
    if handover is None:
        handover = x.numel() // x.shape[-1] >= 32768 and not option_set("NO_FFN_HANDOVER")
    if ln is not None and handover and ffn_ln_train_supported(x, w1, w2):
        gamma, beta, eps, p2, seed2 = ln
        return _FfnLn.apply(x, w1, b1, w2, b2, gamma, beta, eps, drop_p, seed, p2, seed2), None
    scale = 1.0 / (1.0 - drop_p) if drop_p > 0 else 1.0
    h, xa = linear(x, w1, b1, act=1, drop_p=drop_p, seed=seed, with_alias=True, pregated=handover)
    if ln is not None and linear_ln_supported(h, w2, xa):
        gamma, beta, eps, p2, seed2 = ln
        return linear_ln(h, w2, b2, xa, gamma, beta, eps, p2, seed2, in_gate_scale=scale if handover else None), None
    return linear(h, w2, b2, in_gate_scale=scale if handover else None), xa


# ------------------------------------------------------------------------------------------------ sigmoid-gate update
class _GateUpdate(torch.autograd.Function):
    """y = x + u * (sigmoid(z) * keep * scale) in one kernel each way (u None: u is x).  The gate is recomputed from z and the
    keep mask in the backward, nothing else is stored."""

    @staticmethod
    def forward(ctx, x, u, z, keep, scale):
        x, z = _f32c(x, "x"), _f32c(z, "z")
        uu = x if u is None else _f32c(u, "u")
        if uu.shape != x.shape or z.shape != x.shape or (keep is not None and (keep.shape != x.shape or keep.dtype != torch.uint8
                                                                                 or not keep.is_contiguous())):
            raise ValueError("gate update: x, u, z and the keep mask (uint8, contiguous) must have one shape")
        y = torch.empty_like(x)
        _lib.call("mbvae_gate_fwd", x.data_ptr(), uu.data_ptr(), z.data_ptr(), _ptr(keep), float(scale), y.data_ptr(), x.numel(),
                  _stream())
        ctx.save_for_backward(uu, z, keep)
        ctx.cfg = (float(scale), u is None)
        return y

    @staticmethod
    def backward(ctx, dy):
        uu, z, keep = ctx.saved_tensors
        scale, u_is_x = ctx.cfg
        dy = _f32c(dy, "dy")
        du, dz = torch.empty_like(uu), torch.empty_like(z)
        _lib.call("mbvae_gate_bwd", dy.data_ptr(), uu.data_ptr(), z.data_ptr(), _ptr(keep), scale, du.data_ptr(), dz.data_ptr(),
                  uu.numel(), int(u_is_x), _stream())
        return (du, None, dz, None, None) if u_is_x else (dy, du, dz, None, None)


def gate_update(x, u, z, drop_p=0.0, training=False):
    """x + u * dropout(sigmoid(z)) (u None: x + x * dropout(sigmoid(z))): the gated residual updates of TransformerEncoder and
    CrossAttentionFusion (mb_vae_dti/training/models/blocks.py:125, :318-322).  The keep mask is drawn by torch's generator
    (one byte per element), so a captured HIP graph draws fresh masks on every replay."""
    keep, scale = None, 1.0
    if training and drop_p > 0:
        keep = torch.empty(z.shape, dtype=torch.uint8, device=z.device).bernoulli_(1.0 - drop_p)
        scale = 1.0 / (1.0 - drop_p)
    return _GateUpdate.apply(x, u, z, keep, scale)


# ------------------------------------------------------------------------------------------------ gated residual norm
GATED_NORM_MAX_WIDTH = 8192          # columns of a row that one block's registers hold


def gated_residual_norm(x, u=None, z=None, keep=None, keep_scale=1.0, post=None, res_scale=None, pre=None, norm="layer", eps=1e-5):
    """What a residual block does around its products, in one kernel each way:

        v = N_post(u),  y = x + res_scale * sigmoid(z) * keep * keep_scale * v,  n = N_pre(y)        -> (y, n), n None without `pre`

    x, u, z [..., D] of one type (float32, bfloat16, float16), rows may be strided (halves of one projection's output); u None: x
    itself is gated.  z None: no gate.  keep: dropout mask (uint8 or bool, x's shape); where it is 0 nothing is added, whatever u and z
    hold.  post / pre: (gamma, beta) or (gamma, None) of the norm behind the block and of the one that opens the next; None: absent.
    res_scale: [D].  gamma, beta and res_scale share one type, float32 or any other of the three.  norm: "layer" or "rms".  Sums, statistics
    and intermediate values are float32, outputs are rounded once (n comes from the unrounded y); a row whose sum of squares is beyond
    float32 normalises to 0, as in ln_residual.  1 <= D <= 8192.  The gate and
    norm of mb_vae_dti/training/models/blocks.py:92-129, :318-328 (gate_update and ln_residual are the separate forms)."""
    if norm != "layer" and norm != "rms":
        raise ValueError(f"gated_residual_norm: norm is 'layer' or 'rms', got {norm!r}")
    post_g, post_b = post if post is not None else (None, None)
    pre_g, pre_b = pre if pre is not None else (None, None)
    if (post is not None and post_g is None) or (pre is not None and pre_g is None):
        raise ValueError("gated_residual_norm: a norm needs its gamma")
    return _lib.host().gated_residual_norm(x, u, z, keep, keep_scale, post_g, post_b, res_scale, pre_g, pre_b, norm == "rms", eps)


# ------------------------------------------------------------------------------------------------ edge-tensor fan-out
class _EdgeInput(torch.autograd.Function):
    """The three consumers of a layer's edge tensor E in one autograd node: the fused e_mul|e_add projection, the
    Etoy pooling statistics and the residual branch (an alias of E).  Their three gradients would otherwise meet in
    two element-wise accumulation passes over [bs,n,n,de]; here the residual gradient rides in the projection's
    input-gradient epilogue and the pooling gradient is accumulated by its own kernel."""

    @staticmethod
    def forward(ctx, E, w, b, mask, n_nodes):
        E = _f32c(E, "E")
        w = _f32c(w, "weight")
        x2 = E.reshape(-1, E.shape[-1])
        M, K = x2.shape
        N = w.shape[0]
        m8 = _mask_u8(mask)
        ws = workspace(E.device)
        y = torch.empty((M, N), dtype=torch.float32, device=E.device)
        _lib.call("mbvae_linear_fwd", x2.data_ptr(), K, w.data_ptr(), _ptr(b), y.data_ptr(), N, M, K, N, 0,
                  m8.data_ptr(), MASK_EDGE, n_nodes, 0.0, 0, 0, ws.data_ptr(), ws.numel(), _stream(), tag=(M, K, N))
        bs, D = E.shape[0], E.shape[-1]
        L = E.numel() // (bs * D)
        stats = torch.empty((bs, 4 * D), dtype=torch.float32, device=E.device)
        arg = torch.empty((bs, 2, D), dtype=torch.int32, device=E.device)
        _lib.call("mbvae_pool_stats_fwd", E.data_ptr(), stats.data_ptr(), arg.data_ptr(), bs, L, D, _stream())
        ctx.save_for_backward(E, w, m8, stats, arg)
        ctx.cfg = (n_nodes, b is not None)
        return y.reshape(*E.shape[:-1], N), stats, E.view_as(E)

    @staticmethod
    def backward(ctx, dy, dstats, dres):
        E, w, m8, stats, arg = ctx.saved_tensors
        n_nodes, has_bias = ctx.cfg
        dE, dw, db = _edge_input_grads(E, w, m8, stats, arg, n_nodes, has_bias, dy, dstats, dres,
                                       ctx.needs_input_grad[0], ctx.needs_input_grad[1])
        return dE, dw, db, None, None


def _edge_input_grads(E, w, m8, stats, arg, n_nodes, has_bias, dy, dstats, dres, need_dE, need_dw):
    """Gradients of the projection (dy), the pooling statistics (dstats) and the residual alias (dres) w.r.t. E, and
    of the projection w.r.t. its weight and bias."""
    x2 = E.reshape(-1, E.shape[-1])
    M, K = x2.shape
    N = w.shape[0]
    bs, D = E.shape[0], E.shape[-1]
    L = E.numel() // (bs * D)
    ws = workspace(E.device)
    st = _stream()
    dE = dw = db = None
    bf16 = dy is not None and dy.dtype == torch.bfloat16        # bf16 storage mode: the projection output's gradient
    dy2 = (dy.contiguous() if bf16 else _f32c(dy, "dy")).reshape(M, N) if dy is not None else None
    if need_dE and need_dw and dy2 is not None and not bf16 and K == 64 and N == 512:
        # both gradients from one pass over dy (the widest projection: its 2 KB rows are the largest stream of the step)
        dres = _f32c(dres, "dres") if dres is not None else None
        dE = torch.empty_like(E)
        dw = torch.empty((N, K), dtype=torch.float32, device=E.device)
        db = torch.empty((N,), dtype=torch.float32, device=E.device) if has_bias else None
        both = _lib.call("mbvae_linear_bwd_both", dy2.data_ptr(), N, w.data_ptr(), x2.data_ptr(), K, _ptr(dres), dE.data_ptr(), K,
                         dw.data_ptr(), _ptr(db), M, K, N, m8.data_ptr(), MASK_EDGE, n_nodes, ws.data_ptr(), ws.numel(), st,
                         tag=(M, K, N), allow_unsupported=True)
        if both:
            if dstats is not None:
                _lib.call("mbvae_pool_stats_bwd", E.data_ptr(), stats.data_ptr(), arg.data_ptr(), _f32c(dstats).data_ptr(),
                          dE.data_ptr(), bs, L, D, 1, st)
            return dE, dw, db
        dE = dw = db = None
    if need_dE:
        dE = torch.empty_like(E)
        have = False
        if bf16:
            dres = _f32c(dres, "dres") if dres is not None else None
            _lib.call("mbvae_linear_bwd_input_bf16", dy2.data_ptr(), 1, N, w.data_ptr(), _ptr(dres), dE.data_ptr(), 0, K,
                      M, K, N, m8.data_ptr(), MASK_EDGE, n_nodes, st, tag=(M, K, N))
        elif dy2 is not None:
            if dres is not None:
                dres = _f32c(dres, "dres")
                have = _lib.call("mbvae_linear_bwd_input_add", dy2.data_ptr(), N, w.data_ptr(), dres.data_ptr(), dE.data_ptr(),
                                 K, M, K, N, 0, 1.0, m8.data_ptr(), MASK_EDGE, n_nodes, st, tag=(M, K, N),
                                 allow_unsupported=True)
            if not have:
                _lib.call("mbvae_linear_bwd_input", dy2.data_ptr(), N, w.data_ptr(), dE.data_ptr(), K, M, K, N, 0, 1.0,
                          m8.data_ptr(), MASK_EDGE, n_nodes, 0, ws.data_ptr(), ws.numel(), st, tag=(M, K, N))
                if dres is not None:
                    dE += dres
        elif dres is not None:
            dE.copy_(dres)
        else:
            dE.zero_()
        if dstats is not None:
            _lib.call("mbvae_pool_stats_bwd", E.data_ptr(), stats.data_ptr(), arg.data_ptr(), _f32c(dstats).data_ptr(),
                      dE.data_ptr(), bs, L, D, 1, st)
    if need_dw and dy2 is not None:
        dw = torch.empty((N, K), dtype=torch.float32, device=E.device)
        db = torch.empty((N,), dtype=torch.float32, device=E.device) if has_bias else None
        if bf16:
            _lib.call("mbvae_linear_bwd_weight_bf16", dy2.data_ptr(), 1, N, x2.data_ptr(), 0, K, dw.data_ptr(), _ptr(db),
                      M, K, N, m8.data_ptr(), MASK_EDGE, n_nodes, ws.data_ptr(), ws.numel(), st, tag=(M, K, N))
        else:
            _lib.call("mbvae_linear_bwd_weight", dy2.data_ptr(), N, x2.data_ptr(), K, dw.data_ptr(), _ptr(db), M, K, N,
                      0, 1.0, m8.data_ptr(), MASK_EDGE, n_nodes, 0, ws.data_ptr(), ws.numel(), st, tag=(M, K, N))
    return dE, dw, db


def edge_input(E, weight, bias, node_mask, n_nodes):
    """(edge-masked E @ weight^T + bias, pooling statistics of E [bs, 4*de], alias of E for the residual branch)."""
    return _EdgeInput.apply(E, weight, bias, node_mask, n_nodes)


# ------------------------------------------------------------------------------------------------ edge attention
class _EdgeAttention(torch.autograd.Function):
    """QKV [bs,n,3dx] = q|k|v and E12 [bs,n,n,2dx] = e_mul|e_add projection outputs (column blocks, read in place)."""

    @staticmethod
    def forward(ctx, QKV, E12, ye_add, ye_mul, mask, n_head):
        QKV, E12, ye_add, ye_mul = (_f32c(t) for t in (QKV, E12, ye_add, ye_mul))
        bs, n, dx3 = QKV.shape
        dx = dx3 // 3
        scale = 1.0 / math.sqrt(dx // n_head)
        m8 = _mask_u8(mask)
        P = torch.empty((bs, n, n, dx), dtype=torch.float32, device=QKV.device)
        wV = torch.empty((bs, n, dx), dtype=torch.float32, device=QKV.device)
        lse = torch.empty_like(wV)
        q, e = QKV.data_ptr(), E12.data_ptr()
        _lib.call("mbvae_edge_attn_fwd", q, q + 4 * dx, q + 8 * dx, 3 * dx, e, e + 4 * dx, 2 * dx,
                  ye_add.data_ptr(), ye_mul.data_ptr(), m8.data_ptr(), P.data_ptr(), wV.data_ptr(), lse.data_ptr(),
                  bs, n, dx, scale, _stream())
        ctx.save_for_backward(QKV, E12, ye_mul, m8, wV, lse)
        ctx.scale = scale
        ctx.mark_non_differentiable(lse)
        return P, wV, lse

    @staticmethod
    def backward(ctx, dP, dwV, _dlse):
        QKV, E12, ye_mul, m8, wV, lse = ctx.saved_tensors
        dQKV, dE12, dya, dym = _edge_attn_grads(QKV, E12, ye_mul, m8, wV, lse, ctx.scale, dP, dwV)
        return dQKV, dE12, dya, dym, None, None


def _edge_attn_grads(QKV, E12, ye_mul, m8, wV, lse, scale, dP, dwV):
    bs, n, dx = wV.shape
    bf16 = E12.dtype == torch.bfloat16               # bf16 storage mode: E12, dP and dE12 are bf16 in memory
    if dP is None:
        dP = torch.zeros((bs, n, n, dx), dtype=E12.dtype, device=wV.device)
    elif bf16:
        dP = dP.to(torch.bfloat16).contiguous()
    else:
        dP = _f32c(dP)
    dwV = _f32c(dwV) if dwV is not None else torch.zeros_like(wV)
    dE12 = torch.empty_like(E12)
    dQKV = torch.empty_like(QKV)
    dya, dym = torch.empty_like(ye_mul), torch.empty_like(ye_mul)
    q, e, dq, de = QKV.data_ptr(), E12.data_ptr(), dQKV.data_ptr(), dE12.data_ptr()
    es = 2 if bf16 else 4                            # bytes per E12 element: e_add's column block starts dx elements in
    ws = workspace(wV.device)
    _lib.call("mbvae_edge_attn_bwd_bf16" if bf16 else "mbvae_edge_attn_bwd", q, q + 4 * dx, q + 8 * dx, 3 * dx,
              e, e + es * dx, 2 * dx,
              ye_mul.data_ptr(), m8.data_ptr(), wV.data_ptr(), lse.data_ptr(), dP.data_ptr(), dwV.data_ptr(),
              de, de + es * dx, dq, dq + 4 * dx, dq + 8 * dx, dya.data_ptr(), dym.data_ptr(), bs, n, dx, scale,
              ws.data_ptr(), ws.numel(), _stream())
    return dQKV, dE12, dya, dym


def edge_attention(QKV, E12, ye_add, ye_mul, node_mask, n_head):
    """(P, wV): P = ye_add + (ye_mul+1)*Y (input of e_out), wV = per-channel-softmax-weighted values.

    QKV [bs,n,3dx] holds the q|k|v projections side by side, E12 [bs,n,n,2dx] the e_mul|e_add projections."""
    P, wV, _ = _EdgeAttention.apply(QKV, E12, ye_add, ye_mul, node_mask, n_head)
    return P, wV


class _EdgeBlock(torch.autograd.Function):
    """_EdgeInput and _EdgeAttention as ONE node whose forward runs the e_mul|e_add projection inside the attention
    kernel (mbvae_edge_fused_fwd): without gradients the [bs,n,n,2dx] projection output is never written, with
    gradients it is written once (for the backward kernels) but not read back by the forward.  Shapes the fused
    kernel does not take run the two separate forward kernels; the backward is the same either way."""

    @staticmethod
    def forward(ctx, E, w, b, QKV, ye_add, ye_mul, mask, n_head, order=None, pack=None):
        E, w, QKV, ye_add, ye_mul = (_f32c(t) for t in (E, w, QKV, ye_add, ye_mul))
        bs, n = E.shape[0], E.shape[1]
        dx, de = QKV.shape[-1] // 3, E.shape[-1]
        M, N = bs * n * n, 2 * dx
        scale = 1.0 / math.sqrt(dx // n_head)
        m8 = _mask_u8(mask)
        dev = E.device
        need_grad = any(ctx.needs_input_grad[:6])
        if pack is not None and (need_grad or order is None or not order.sparse):
            raise RuntimeError("packed node rows are an inference-only layout (sparse row order, no gradients)")
        # bf16 storage mode: P and E1|E2 leave the fused kernel as bf16 (training form, fused shapes only)
        store = torch.bfloat16 if (_BF16_STORAGE and need_grad and de == 64 and dx == 256 and n <= 64) else torch.float32
        P = torch.empty((bs, n, n, dx), dtype=store, device=dev)
        if pack is None:
            wV = torch.empty((bs, n, dx), dtype=torch.float32, device=dev)
        else:                           # packed rows; the padding row is never written by the kernel and must be finite
            wV = torch.zeros((QKV.shape[0], dx), dtype=torch.float32, device=dev)
        lse = torch.empty_like(wV)
        q = QKV.data_ptr()
        # training, fp32: first choice is the forward that does NOT store E1|E2 (the backward recomputes it from E)
        recompute = False
        if need_grad and pack is None:
            recompute = _lib.call("mbvae_edge_fused_fwd_recompute_bf16" if store == torch.bfloat16 else "mbvae_edge_fused_fwd_recompute",
                                  E.data_ptr(), w.data_ptr(), _ptr(b), q, q + 4 * dx, q + 8 * dx,
                                  3 * dx, ye_add.data_ptr(), ye_mul.data_ptr(), m8.data_ptr(), P.data_ptr(), wV.data_ptr(),
                                  lse.data_ptr(), bs, n, de, dx, scale, _stream(), allow_unsupported=True)
        E12 = torch.empty((bs, n, n, N), dtype=store, device=dev) if (need_grad and not recompute) else None
        if recompute:
            fused = True
        elif store == torch.bfloat16:
            _lib.call("mbvae_edge_fused_fwd_bf16", E.data_ptr(), w.data_ptr(), _ptr(b), q, q + 4 * dx, q + 8 * dx, 3 * dx,
                      ye_add.data_ptr(), ye_mul.data_ptr(), m8.data_ptr(), P.data_ptr(), wV.data_ptr(), lse.data_ptr(),
                      E12.data_ptr(), bs, n, de, dx, scale, _stream())
            fused = True
        else:
            fused = _lib.call("mbvae_edge_fused_fwd", E.data_ptr(), w.data_ptr(), _ptr(b), q, q + 4 * dx, q + 8 * dx, 3 * dx,
                              ye_add.data_ptr(), ye_mul.data_ptr(), m8.data_ptr(), P.data_ptr(), wV.data_ptr(), lse.data_ptr(),
                              _ptr(E12), 0 if need_grad else _work_counter(dev).data_ptr(),
                              0 if pack is None else pack.off.data_ptr(), 0 if pack is None else pack.by_size.data_ptr(),
                              bs, n, de, dx, scale, _stream(), allow_unsupported=True)
        if not fused and pack is not None:
            raise RuntimeError("packed node rows need the fused attention kernel (de = 64, dx = 256, n <= 64)")
        if not fused:
            if E12 is None:
                E12 = torch.empty((bs, n, n, N), dtype=torch.float32, device=dev)
            ws = workspace(dev)
            _lib.call("mbvae_linear_fwd", E.data_ptr(), de, w.data_ptr(), _ptr(b), E12.data_ptr(), N, M, de, N, 0,
                      m8.data_ptr(), MASK_EDGE, n, 0.0, 0, 0, ws.data_ptr(), ws.numel(), _stream(), tag=(M, de, N))
            e = E12.data_ptr()
            _lib.call("mbvae_edge_attn_fwd", q, q + 4 * dx, q + 8 * dx, 3 * dx, e, e + 4 * dx, N,
                      ye_add.data_ptr(), ye_mul.data_ptr(), m8.data_ptr(), P.data_ptr(), wV.data_ptr(), lse.data_ptr(),
                      bs, n, dx, scale, _stream())
        if order is not None and order.sparse and not need_grad:
            stats = pool_stats_pairs(E, order)       # E's padding rows are not all written: pool the valid pairs
            arg = None
        else:
            stats = torch.empty((bs, 4 * de), dtype=torch.float32, device=dev)
            arg = torch.empty((bs, 2, de), dtype=torch.int32, device=dev)
            _lib.call("mbvae_pool_stats_fwd", E.data_ptr(), stats.data_ptr(), arg.data_ptr(), bs, n * n, de, _stream())
        if need_grad:
            ctx.save_for_backward(E, w, m8, stats, arg, QKV, E12, ye_mul, wV, lse, b)
        ctx.cfg = (n, b is not None, scale)
        ctx.store = store
        return P, wV, stats, E.view_as(E)

    @staticmethod
    def backward(ctx, dP, dwV, dstats, dres):
        E, w, m8, stats, arg, QKV, E12, ye_mul, wV, lse, b = ctx.saved_tensors
        n, has_bias, scale = ctx.cfg
        if E12 is None:                  # the forward did not store E1|E2: gradients from E with the projection recomputed
            bs, dx = E.shape[0], wV.shape[-1]
            bf16 = ctx.store == torch.bfloat16
            if dP is None:
                dP = torch.zeros((bs, n, n, dx), dtype=ctx.store, device=E.device)
            else:
                dP = dP.to(torch.bfloat16).contiguous() if bf16 else _f32c(dP)
            dwV = _f32c(dwV) if dwV is not None else torch.zeros_like(wV)
            dE12 = torch.empty((bs, n, n, 2 * dx), dtype=ctx.store, device=E.device)
            dQKV = torch.empty_like(QKV)
            dya, dym = torch.empty_like(ye_mul), torch.empty_like(ye_mul)
            q, dq = QKV.data_ptr(), dQKV.data_ptr()
            _lib.call("mbvae_edge_fused_bwd_bf16" if bf16 else "mbvae_edge_fused_bwd", E.data_ptr(), w.data_ptr(), _ptr(b), q, q + 4 * dx, q + 8 * dx, 3 * dx,
                      ye_mul.data_ptr(), m8.data_ptr(), wV.data_ptr(), lse.data_ptr(), dP.data_ptr(), dwV.data_ptr(),
                      dE12.data_ptr(), dq, dq + 4 * dx, dq + 8 * dx, dya.data_ptr(), dym.data_ptr(), bs, n, E.shape[-1], dx,
                      scale, _stream())
        else:
            dQKV, dE12, dya, dym = _edge_attn_grads(QKV, E12, ye_mul, m8, wV, lse, scale, dP, dwV)
        dE, dw, db = _edge_input_grads(E, w, m8, stats, arg, n, has_bias, dE12, dstats, dres,
                                       ctx.needs_input_grad[0], ctx.needs_input_grad[1])
        return dE, dw, db, dQKV, dya, dym, None, None, None, None


def edge_block(E, weight, bias, QKV, ye_add, ye_mul, node_mask, n_head, order=None, pack=None):
    """(P, wV, pooling statistics of E, alias of E): edge_input followed by edge_attention, with the projection
    output kept out of memory whenever the fused forward kernel takes the shape.  Without gradients P is only
    written for valid pairs (see zero_masked_pairs_).  order: a sparse EdgeRowOrder says that E's padding rows hold
    one common row of which only the order's first padding tile is actually stored (see EdgeRowOrder).  pack: QKV
    (and the returned wV) hold packed node rows [rows, .] (see NodePack) instead of [bs, n, .]."""
    return _EdgeBlock.apply(E, weight, bias, QKV, ye_add, ye_mul, node_mask, n_head, order, pack)


# ------------------------------------------------------------------------------------------------ residual + LayerNorm
class _LnResidual(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, r, gamma, beta, eps, drop_p, seed):
        x = _f32c(x, "x")
        r = _f32c(r, "r") if r is not None else None
        D = x.shape[-1]
        rows = x.numel() // D
        y = torch.empty_like(x)
        mean = torch.empty(rows, dtype=torch.float32, device=x.device)
        rstd = torch.empty(rows, dtype=torch.float32, device=x.device)
        _lib.call("mbvae_ln_residual_fwd", x.data_ptr(), _ptr(r), gamma.data_ptr(), beta.data_ptr(), y.data_ptr(),
                  mean.data_ptr(), rstd.data_ptr(), rows, D, float(eps), float(drop_p), int(seed), _stream())
        ctx.save_for_backward(x, r, gamma, mean, rstd)
        ctx.cfg = (float(drop_p), int(seed))
        return y

    @staticmethod
    def backward(ctx, dy):
        x, r, gamma, mean, rstd = ctx.saved_tensors
        drop_p, seed = ctx.cfg
        D = x.shape[-1]
        rows = x.numel() // D
        dy = _f32c(dy, "dy")
        dx = torch.empty_like(x)
        dr = torch.empty_like(x) if (r is not None and drop_p > 0) else None
        dgamma, dbeta = torch.empty_like(gamma), torch.empty_like(gamma)
        ws = workspace(x.device)
        _lib.call("mbvae_ln_residual_bwd", x.data_ptr(), _ptr(r), gamma.data_ptr(), mean.data_ptr(), rstd.data_ptr(),
                  dy.data_ptr(), dx.data_ptr(), _ptr(dr), dgamma.data_ptr(), dbeta.data_ptr(), rows, D, drop_p, seed,
                  ws.data_ptr(), ws.numel(), _stream())
        if r is not None and dr is None:
            dr = dx          # no dropout: the residual branch receives the same gradient
        return dx, dr, dgamma, dbeta, None, None, None


class _LinearLn(torch.autograd.Function):
    """LayerNorm(resid + dropout(rowmask(x @ W^T + b))) with the normalisation in the product's epilogue
    (mbvae_linear_ln_fwd): the Linear's output never travels through memory and the backward reads ONE stored tensor
    (the pre-LayerNorm sum) instead of the residual and the Linear's output.  The leading arguments are _Linear's, so
    the Linear's own gradients come from _Linear.backward run on this node's dr."""

    class _LinCtx:                       # what _Linear.backward reads from its ctx
        pass

    @staticmethod
    def forward(ctx, x, w, b, resid, gamma, beta, mask, mask_mode, n_nodes, eps, drop_p, seed, in_gate_scale):
        bf16_in = x.dtype == torch.bfloat16          # bf16 storage mode: the attention output P feeding e_out
        x2 = x.contiguous().reshape(-1, x.shape[-1]) if bf16_in else _f32c(x, "x").reshape(-1, x.shape[-1])
        w, resid, gamma, beta = _f32c(w, "weight"), _f32c(resid, "resid"), _f32c(gamma), _f32c(beta)
        M, K = x2.shape
        N = w.shape[0]
        m8 = _mask_u8(mask)
        y, z = torch.empty_like(resid), torch.empty_like(resid)
        ok = _lib.call("mbvae_linear_ln_fwd_bf16" if bf16_in else "mbvae_linear_ln_fwd", x2.data_ptr(), K, w.data_ptr(), _ptr(b), resid.data_ptr(), gamma.data_ptr(),
                       beta.data_ptr(), y.data_ptr(), z.data_ptr(), M, K, N, _ptr(m8), mask_mode, n_nodes, float(eps),
                       float(drop_p), int(seed), _stream(), tag=(M, K, N), allow_unsupported=True)
        if not ok:
            raise RuntimeError("mbvae_linear_ln_fwd does not take this shape (check linear_ln_supported first)")
        ctx.save_for_backward(x2, w, m8, z, gamma)
        ctx.cfg = (mask_mode, n_nodes, float(eps), float(drop_p), int(seed), b is not None, x.shape, in_gate_scale)
        return y

    @staticmethod
    def backward(ctx, dy):
        x2, w, m8, z, gamma = ctx.saved_tensors
        mask_mode, n_nodes, eps, drop_p, seed, has_bias, xshape, in_gate_scale = ctx.cfg
        D = z.shape[-1]
        rows = z.numel() // D
        dy = _f32c(dy, "dy")
        dres = torch.empty_like(z)
        need_lin = any(ctx.needs_input_grad[:3])
        dr = torch.empty_like(z) if (drop_p > 0 and need_lin) else None
        dgamma, dbeta = torch.empty_like(gamma), torch.empty_like(gamma)
        ws = workspace(z.device)
        _lib.call("mbvae_ln_sum_bwd", z.data_ptr(), gamma.data_ptr(), dy.data_ptr(), dres.data_ptr(), _ptr(dr),
                  dgamma.data_ptr(), dbeta.data_ptr(), rows, D, eps, drop_p, seed, ws.data_ptr(), ws.numel(), _stream())
        dx = dw = db = None
        if need_lin:
            lin = _LinearLn._LinCtx()
            lin.saved_tensors = (x2, w, None, m8)
            lin.cfg = (mask_mode, n_nodes, 0.0, False, has_bias, xshape)
            lin.in_gate_scale, lin.relu = in_gate_scale, False
            lin.needs_input_grad = tuple(ctx.needs_input_grad[:3])
            dx, dw, db = _Linear.backward(lin, dr if dr is not None else dres)[:3]
        return dx, dw, db, dres, dgamma, dbeta, None, None, None, None, None, None, None


def linear_ln_supported(x, weight, resid):
    """Shapes mbvae_linear_ln_fwd takes: a 64-wide fp32 Linear over >= 8192 rows (the edge tensor's e_out and linE2)."""
    M = x.numel() // x.shape[-1]
    K = x.shape[-1]
    return (x.is_cuda and x.dtype in (torch.float32, torch.bfloat16) and weight.shape[0] == 64 and resid.shape[-1] == 64 and K % 64 == 0
            and K <= 384 and M >= 8192 and M % 32 == 0 and M * 64 < 0x3fffffff
            and not (option_set("NO_LN_EPILOGUE") or option_set("NO_TSGEMM") or option_set("NO_TSGEMM2")))


def linear_ln(x, weight, bias, resid, gamma, beta, eps=1e-5, drop_p=0.0, seed=0, mask=None, mask_mode=MASK_NONE, n_nodes=0,
              in_gate_scale=None):
    """LayerNorm(resid + dropout(rowmask(x @ W^T + b))) * gamma + beta in one kernel; see linear_ln_supported.
    in_gate_scale: as for linear() - x came out of a ReLU (+ dropout) layer whose gate this layer's backward applies."""
    if mask is None:
        mask_mode = MASK_NONE
    return _LinearLn.apply(x, weight, bias, resid, gamma, beta, mask, mask_mode, n_nodes, eps, drop_p, seed, in_gate_scale)


def ln_residual(x, r, gamma, beta, eps=1e-5, drop_p=0.0, seed=0):
    """LayerNorm(x + dropout(r)) * gamma + beta over the last dimension (r may be None)."""
    return _LnResidual.apply(x, r, _f32c(gamma), _f32c(beta), eps, drop_p, seed)


def edge_tile_map(node_mask):
    """uint8 [ceil(bs*n*n/32)]: 1 where the tile of 32 consecutive pair rows (b,i,j) holds a valid pair, 0 where all
    of them are padding.  Lets the inference kernels below skip padding tiles of ragged batches (the mask is the same
    for every layer and every reverse-diffusion step)."""
    m = node_mask.bool()
    pair = (m.unsqueeze(1) & m.unsqueeze(2)).reshape(-1)
    pad = -pair.numel() % 32
    if pad:
        pair = torch.cat((pair, pair.new_zeros(pad)))
    return pair.view(-1, 32).any(1).to(torch.uint8)


class EdgeRowOrder:
    """Packed order of the bs*n*n pair rows of a ragged batch for the fused inference kernels: `idx` (int32) lists the
    valid rows (both nodes unmasked) in ascending order, padded to a multiple of 32 by repeating the last one, then
    the padding rows, padded likewise; `nvalid` (int32 [2], on the device) holds the number of valid rows and the
    `sparse` flag.  With sparse=True the kernels evaluate and store only the first padding tile (it carries the
    padding rows' common value from kernel to kernel) and leave the other padding rows of their outputs unwritten:
    the caller must then pool with pool_stats_pairs and call zero_masked_pairs_ before any other consumer.
    Built without a host synchronisation; the node mask must not change while the object is in use."""

    def __init__(self, node_mask, sparse=False):
        m = node_mask.bool()
        pair = (m.unsqueeze(1) & m.unsqueeze(2)).reshape(-1)
        M = pair.numel()
        dev = pair.device
        nv = pair.sum()
        order = torch.argsort(~pair, stable=True)                      # valid rows first, each part ascending
        nvt32 = (nv + 31) // 32 * 32
        pos = torch.arange(M + 64, device=dev)
        src = torch.where(pos < nvt32, torch.minimum(pos, (nv - 1).clamp(min=0)),
                          torch.minimum(nv + pos - nvt32, torch.full_like(nv, M - 1)))
        self.idx = order[src.clamp(min=0)].to(torch.int32).contiguous()
        self.nvalid = torch.stack((nv, torch.full_like(nv, int(sparse)))).to(torch.int32).contiguous()
        self.rows = M
        self.sparse = bool(sparse)
        self.mask_u8 = _mask_u8(node_mask)
        self.n = node_mask.shape[1]


def edge_row_order(node_mask, sparse=False):
    """EdgeRowOrder of a node mask, or None when the batch has fewer than 32 pair rows."""
    bs, n = node_mask.shape
    return EdgeRowOrder(node_mask, sparse) if bs * n * n >= 32 else None


def pool_stats_pairs(E, order):
    """[bs, 4*de] = mean | min | max | unbiased std of E [bs,n,n,de] over all n*n pairs, reading only the valid pairs:
    the padding pairs all hold the row E[order's first padding row] (caller's guarantee) and enter analytically.
    No gradients; raises for widths the kernel does not take (de != 64)."""
    E = _f32c(E, "E")
    bs, n, de = E.shape[0], E.shape[1], E.shape[-1]
    stats = torch.empty((bs, 4 * de), dtype=torch.float32, device=E.device)
    with torch.no_grad():
        if not _lib.call("mbvae_pool_stats_pairs_fwd", E.data_ptr(), stats.data_ptr(), order.mask_u8.data_ptr(),
                         order.idx.data_ptr(), order.nvalid.data_ptr(), bs, n, de, _stream(), allow_unsupported=True):
            raise RuntimeError("pool_stats_pairs: unsupported width for a sparse row order")
    return stats


class NodePack:
    """Packed node rows of a ragged batch for the no-gradient denoiser: `rows` (int64) lists the valid nodes' flat
    indices b*n + i in ascending order followed, if the batch has padding at all, by ONE padding node (row `pad_row`
    of the packed tensors: it carries the value all padding nodes share from op to op); `off` (int32 [bs+1]) are the
    graphs' offsets into the packed rows; `graph` (int64) the graph of each packed row; `keep` (uint8 [1, rows]) is 0
    for the padding row; `by_size` (int32 [bs]) lists the graphs from the largest to the smallest, the order in which
    the attention kernel hands out its per-graph tasks.  Only for masks that keep a prefix of every graph's nodes (None otherwise).  Building it
    synchronises with the host once."""

    @staticmethod
    def build(node_mask):
        m = node_mask.bool()
        bs, n = m.shape
        nb = m.sum(1)
        if not bool((m == (torch.arange(n, device=m.device).unsqueeze(0) < nb.unsqueeze(1))).all()):
            return None
        self = NodePack()
        flat = m.reshape(-1)
        valid = flat.nonzero().flatten()
        pad = (~flat).nonzero().flatten()[:1]
        self.rows = torch.cat((valid, pad)).contiguous()
        self.n_valid = int(valid.numel())
        self.pad_row = self.n_valid if pad.numel() else 0
        self.off = torch.cat((nb.new_zeros(1), nb.cumsum(0))).to(torch.int32).contiguous()
        self.graph = torch.div(self.rows, n, rounding_mode="floor")
        self.by_size = torch.argsort(nb, descending=True, stable=True).to(torch.int32).contiguous()   # largest graphs first
        keep = torch.ones(self.rows.numel(), dtype=torch.uint8, device=m.device)
        if pad.numel():
            keep[-1] = 0
        self.keep = keep.reshape(1, -1)
        self.bs, self.n = bs, n
        return self


def pool_stats_nodes(Xp, pack):
    """[bs, 4*dx] = mean | min | max | unbiased std over all n nodes of every graph from packed rows Xp (NodePack):
    the padding nodes enter as (n - nb) copies of the pack's padding row.  No gradients."""
    Xp = _f32c(Xp, "Xp")
    D = Xp.shape[-1]
    stats = torch.empty((pack.bs, 4 * D), dtype=torch.float32, device=Xp.device)
    _lib.call("mbvae_pool_stats_nodes_fwd", Xp.data_ptr(), stats.data_ptr(), pack.off.data_ptr(), pack.pad_row, pack.bs,
              pack.n, D, _stream())
    return stats


def zero_masked_pairs_(P, node_mask):
    """In place: P[b,i,j,:] = 0 where node i or j is masked.  The no-gradient form of edge_block leaves those rows
    unwritten; every consumer other than the fused e_out kernel (which skips them itself) calls this first."""
    m = node_mask.bool()
    return P.masked_fill_(~(m.unsqueeze(1) & m.unsqueeze(2)).unsqueeze(-1), 0.0)


def _order_args(order, tile_map, rows):
    """(tile_ok, row_idx, nvalid) pointers of the optional padding shortcuts; a row order wins over a tile map."""
    if order is not None:
        if order.rows != rows:
            raise ValueError("row order does not match the number of rows")
        return 0, order.idx.data_ptr(), order.nvalid.data_ptr()
    if tile_map is not None and tile_map.numel() != (rows + 31) // 32:
        raise ValueError("tile_map does not match the number of rows")
    return _ptr(tile_map), 0, 0


def ffn_ln_inference(x, w1, b1, w2, b2, gamma, beta, eps=1e-5, tile_map=None, order=None):
    """LayerNorm(x + linear(relu(linear(x, w1, b1)), w2, b2)) * gamma + beta without gradients or dropout.
    One fused kernel where the widths allow (64 -> 128 -> 64), else the three separate kernels.
    tile_map (edge_tile_map): tiles marked 0 must consist of padding rows that all hold the same values; one of them
    is evaluated and copied to the rest (same bits as evaluating each).  order (edge_row_order): the same guarantee
    for the padding rows, and the valid rows are packed into whole tiles."""
    x = _f32c(x, "x")
    d, dff = x.shape[-1], w1.shape[0]
    rows = x.numel() // d
    tm, ri, nvp = _order_args(order, tile_map, rows)
    with torch.no_grad():
        out = torch.empty_like(x)
        if _lib.call("mbvae_edge_ffn_fwd", x.data_ptr(), _f32c(w1).data_ptr(), _ptr(b1), _f32c(w2).data_ptr(), _ptr(b2),
                     _f32c(gamma).data_ptr(), _f32c(beta).data_ptr(), out.data_ptr(), tm, ri, nvp, rows, d, dff,
                     float(eps), _stream(), allow_unsupported=True):
            return out
        return ln_residual(x, linear(linear(x, w1, b1, act=1), w2, b2), gamma, beta, eps)


def edge_out_ln_inference(P, w, b, E, node_mask, n_nodes, gamma, beta, eps=1e-5, tile_map=None, order=None,
                          uniform_padding=False):
    """LayerNorm(E + edge_mask * linear(P, w, b)) * gamma + beta without gradients or dropout: one fused kernel
    where the widths allow (256 -> 64), else the projection and the residual LayerNorm kernels.
    P is only read on valid pairs (it may be uninitialised elsewhere); tile_map (edge_tile_map) or order
    (edge_row_order) let whole padding tiles go unfetched; uniform_padding: every padding row of E holds the same
    values, so one is normalised and copied to the rest."""
    P, E = _f32c(P, "P"), _f32c(E, "E")
    dx, de = P.shape[-1], E.shape[-1]
    rows = E.numel() // de
    tm, ri, nvp = _order_args(order, tile_map, rows)
    with torch.no_grad():
        out = torch.empty_like(E)
        m8 = _mask_u8(node_mask)
        if _lib.call("mbvae_edge_out_ln_fwd", P.data_ptr(), _f32c(w).data_ptr(), _ptr(b), E.data_ptr(), m8.data_ptr(),
                     n_nodes, _f32c(gamma).data_ptr(), _f32c(beta).data_ptr(), out.data_ptr(), tm, ri, nvp,
                     int(bool(uniform_padding)), rows, dx, de, float(eps), _stream(), allow_unsupported=True):
            return out
        P = zero_masked_pairs_(P.view(-1, n_nodes, n_nodes, dx), node_mask).view_as(P)
        return ln_residual(E, linear(P, w, b, mask=node_mask, mask_mode=MASK_EDGE, n_nodes=n_nodes), gamma, beta, eps)


# ------------------------------------------------------------------------------------------------ pooling
class _PoolStats(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x):
        x = _f32c(x, "x")
        bs, D = x.shape[0], x.shape[-1]
        L = x.numel() // (bs * D)
        stats = torch.empty((bs, 4 * D), dtype=torch.float32, device=x.device)
        arg = torch.empty((bs, 2, D), dtype=torch.int32, device=x.device)
        _lib.call("mbvae_pool_stats_fwd", x.data_ptr(), stats.data_ptr(), arg.data_ptr(), bs, L, D, _stream())
        ctx.save_for_backward(x, stats, arg)
        return stats

    @staticmethod
    def backward(ctx, dstats):
        x, stats, arg = ctx.saved_tensors
        bs, D = x.shape[0], x.shape[-1]
        L = x.numel() // (bs * D)
        dx = torch.empty_like(x)
        _lib.call("mbvae_pool_stats_bwd", x.data_ptr(), stats.data_ptr(), arg.data_ptr(), _f32c(dstats).data_ptr(),
                  dx.data_ptr(), bs, L, D, 0, _stream())
        return dx


def pool_stats(x):
    """x [bs, ..., D] -> [bs, 4D] = mean | min | max | unbiased std over the middle dimensions."""
    return _PoolStats.apply(x)


# ------------------------------------------------------------------------------------------------ symmetrise + mask
class _SymMask(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, skip, mask, zero_diag):
        x = _f32c(x, "x")
        bs, n, _, D = x.shape
        m8 = _mask_u8(mask)
        out = torch.empty_like(x)
        lds = 0
        if skip is not None:
            skip = _f32c(skip, "skip")
            lds = skip.shape[-1]
        _lib.call("mbvae_sym_mask", x.data_ptr(), _ptr(skip), lds, m8.data_ptr(), out.data_ptr(), bs, n, D,
                  int(zero_diag), _stream())
        ctx.save_for_backward(m8)
        ctx.zero_diag = int(zero_diag)
        ctx.skip_width = lds
        return out

    @staticmethod
    def backward(ctx, dout):
        (m8,) = ctx.saved_tensors
        dout = _f32c(dout)
        bs, n, _, D = dout.shape
        dx = torch.empty_like(dout)
        _lib.call("mbvae_sym_mask", dout.data_ptr(), 0, 0, m8.data_ptr(), dx.data_ptr(), bs, n, D, ctx.zero_diag, _stream())
        dskip = None
        if ctx.needs_input_grad[1]:          # the skip input normally is data; only parity tests ask for this
            dskip = dx.new_zeros(bs, n, n, ctx.skip_width)
            dskip[..., :D] = dx
        return dx, dskip, None, None


def sym_mask(x, node_mask, skip=None, zero_diag=False):
    """0.5*(x + x^T (+ skip + skip^T)) * pair mask (* off-diagonal).  `skip` contributes its first D features."""
    return _SymMask.apply(x, skip, node_mask, zero_diag)


# ------------------------------------------------------------------------------------------------ FiLM of the node update
class _Film(torch.autograd.Function):
    @staticmethod
    def forward(ctx, add, mul, x):
        add, mul, x = _f32c(add, "add"), _f32c(mul, "mul"), _f32c(x, "x")
        bs, n, D = x.shape
        out = torch.empty_like(x)
        _lib.call("mbvae_film_fwd", add.data_ptr(), mul.data_ptr(), x.data_ptr(), out.data_ptr(), bs, n, D, _stream())
        ctx.save_for_backward(mul, x)
        return out

    @staticmethod
    def backward(ctx, dout):
        mul, x = ctx.saved_tensors
        bs, n, D = x.shape
        dout = _f32c(dout, "dout")
        dx = torch.empty_like(x)
        dadd, dmul = torch.empty_like(mul), torch.empty_like(mul)
        _lib.call("mbvae_film_bwd", dout.data_ptr(), mul.data_ptr(), x.data_ptr(), dx.data_ptr(), dadd.data_ptr(), dmul.data_ptr(),
                  bs, n, D, _stream())
        return dadd, dmul, dx


def film(add, mul, x):
    """add[:, None] + (mul[:, None] + 1) * x for x [bs,n,D], add / mul [bs,D] (graph_transformer.py:254) in one kernel
    each way (the torch expression is three launches forward and five backward)."""
    return _Film.apply(add, mul, x)


# ------------------------------------------------------------------------------------------------ losses
CE_SLOTS = 18


class _MaskedCE(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, target):
        logits, target = _f32c(logits, "logits"), _f32c(target, "target")
        C = logits.shape[-1]
        rows = logits.numel() // C
        out = torch.empty(CE_SLOTS, dtype=torch.float32, device=logits.device)
        ws = workspace(logits.device)
        _lib.call("mbvae_masked_ce_fwd", logits.data_ptr(), target.data_ptr(), out.data_ptr(), rows, C, ws.data_ptr(),
                  ws.numel(), _stream())
        ctx.save_for_backward(logits, target, out)
        loss = out[0] / out[1].clamp(min=1.0)
        stats = out.detach()
        ctx.mark_non_differentiable(stats)
        return loss, stats

    @staticmethod
    def backward(ctx, dloss, _dstats):
        logits, target, out = ctx.saved_tensors
        C = logits.shape[-1]
        rows = logits.numel() // C
        coef = (dloss / out[1].clamp(min=1.0)).reshape(1).float().contiguous()
        dlogits = torch.empty_like(logits)
        _lib.call("mbvae_masked_ce_bwd", logits.data_ptr(), target.data_ptr(), coef.data_ptr(), dlogits.data_ptr(), rows, C,
                  _stream())
        return dlogits, None


def masked_ce(logits, target):
    """(mean CE over rows whose one-hot target is non-zero, stats) with stats = [sum CE, #rows, per-class BCE sums...]."""
    return _MaskedCE.apply(logits, target)


class _KLReparam(torch.autograd.Function):
    @staticmethod
    def forward(ctx, mu, logvar, eps):
        mu, logvar, eps = _f32c(mu), _f32c(logvar), _f32c(eps)
        z = torch.empty_like(mu)
        kl = torch.empty(1, dtype=torch.float32, device=mu.device)
        ws = workspace(mu.device)
        _lib.call("mbvae_kl_reparam_fwd", mu.data_ptr(), logvar.data_ptr(), eps.data_ptr(), z.data_ptr(), kl.data_ptr(),
                  mu.numel(), ws.data_ptr(), ws.numel(), _stream())
        ctx.save_for_backward(mu, logvar, eps)
        return z, kl.reshape(())

    @staticmethod
    def backward(ctx, dz, dkl):
        mu, logvar, eps = ctx.saved_tensors
        dmu, dlv = torch.empty_like(mu), torch.empty_like(mu)
        dz = _f32c(dz) if dz is not None else None
        dkl = dkl.reshape(1).float().contiguous() if dkl is not None else None
        _lib.call("mbvae_kl_reparam_bwd", mu.data_ptr(), logvar.data_ptr(), eps.data_ptr(), _ptr(dz), _ptr(dkl),
                  dmu.data_ptr(), dlv.data_ptr(), mu.numel(), _stream())
        return dmu, dlv, None


def kl_reparam(mu, logvar, eps):
    """(z, kl): z = mu + eps*exp(logvar/2); kl = -0.5*mean(1 + logvar - mu^2 - exp(logvar))."""
    return _KLReparam.apply(mu, logvar, eps)


# ------------------------------------------------------------------------------------------------ eigensolver
@torch.no_grad()
def sym_eig(A):
    """Batched symmetric eigendecomposition A [bs,n,n] (n <= 64) -> (W ascending [bs,n], V [bs,n,n] columns)."""
    A = _f32c(A, "A")
    bs, n, _ = A.shape
    W = torch.empty((bs, n), dtype=torch.float32, device=A.device)
    V = torch.empty_like(A)
    _lib.call("mbvae_sym_eig", A.data_ptr(), W.data_ptr(), V.data_ptr(), bs, n, _stream())
    return W, V


# ------------------------------------------------------------------------------------------------ class-id wire format
@torch.no_grad()
def dense_from_ids(atom_ids, bond_ids, cx, ce):
    """int8 class ids (atoms [bs,n], < 0 = padding; bonds [bs,n,n], 0 = none) -> (X one-hot [bs,n,cx],
    E one-hot [bs,n,n,ce], node_mask bool [bs,n]) in the dense-batch convention (unmasked, class 0 on every
    bond-less off-diagonal pair, zero diagonal)."""
    if not atom_ids.is_cuda or atom_ids.dtype != torch.int8 or bond_ids.dtype != torch.int8:
        raise RuntimeError("dense_from_ids: expected int8 class-id tensors on the GPU; the HIP path has no CPU fallback")
    atom_ids, bond_ids = atom_ids.contiguous(), bond_ids.contiguous()
    bs, n = atom_ids.shape
    X = torch.empty((bs, n, cx), dtype=torch.float32, device=atom_ids.device)
    E = torch.empty((bs, n, n, ce), dtype=torch.float32, device=atom_ids.device)
    mask = torch.empty((bs, n), dtype=torch.uint8, device=atom_ids.device)
    _lib.call("mbvae_dense_from_ids", atom_ids.data_ptr(), bond_ids.data_ptr(), X.data_ptr(), E.data_ptr(), mask.data_ptr(),
              bs, n, cx, ce, _stream())
    return X, E, mask.view(torch.bool)


# ------------------------------------------------------------------------------------------------ embedding
def embedding(ids, weight, scale=1.0):
    """scale * weight[ids]: rows of a table by class id, ids of any shape (int8, int16, uint8, int32, int64), weight [V, D] (float32,
    bfloat16, float16) -> [*ids.shape, D].  Ids outside [0, V) - the -1 of padding in the class-id wire format - give a row of zeros and
    take no gradient.  The table's gradient sums the rows of equal ids in float32, in an order that the ids alone decide."""
    return _lib.host().embedding(ids, weight, scale)


# ------------------------------------------------------------------------------------------------ gradient norm and clipping
def global_grad_norm(grads, norm_type=2.0):
    """(sum |g|^p)^(1/p) over all values of a list of gradients (None entries are skipped), p = 1, 2 or infinity: one float32 value on
    the GPU, without a host synchronisation.  Sums are float64."""
    grads = [g for g in grads if g is not None]
    if not grads:
        return torch.zeros((), device="cuda")
    return _lib.host().grad_clip(grads, [], -1.0, norm_type)


def clip_grad_norm_(grads, max_norm, norm_type=2.0, out=None):
    """Scales a list of gradients (p.grad of a model's parameters; None entries are skipped) by min(1, max_norm / (norm + 1e-6)) and
    returns their norm before it as one float32 value on the GPU: what Lightning's gradient_clip_val does (mb_vae_dti/training/run.py:638-654).
    In place, or into `out`: as many tensors of the same types and layouts.  float32, bfloat16 and float16 may be mixed.  Where norm + 1e-6
    <= max_norm, or max_norm is infinity, the values stay bit for bit.  The factor comes from the float64 norm: one beyond float32 is
    returned as infinity and still scales by what it is.  Where a value is infinite the factor is 0, where one is NaN every gradient becomes
    NaN.  No tensor may share memory with another one that is written."""
    grads, outs = list(grads), None if out is None else list(out)
    if outs is not None and len(outs) != len(grads):
        raise ValueError(f"clip_grad_norm_: {len(grads)} gradients, but {len(outs)} outputs")
    if not max_norm >= 0:
        raise ValueError(f"clip_grad_norm_: max_norm must not be negative, got {max_norm}")
    if outs is not None:
        outs = [o for o, g in zip(outs, grads) if g is not None]
        if any(o is None for o in outs):
            raise ValueError("clip_grad_norm_: an output is missing for one of the gradients")
    grads = [g for g in grads if g is not None]
    if not grads:
        return torch.zeros((), device="cuda")
    return _lib.host().grad_clip(grads, outs or [], max_norm, norm_type)


def clip_grad_norm_takes(grads):
    """Whether clip_grad_norm_ takes these gradients: dense float32, bfloat16 or float16 tensors on one GPU that ask for no gradient themselves."""
    return _lib.host().grad_clip_takes([g for g in grads if g is not None])


# ------------------------------------------------------------------------------------------------ diffusion samplers
@torch.no_grad()
def apply_noise(X0, E0, node_mask, abar_t, mx, me, expX, expE):
    """Forward-noise one batch.  Returns (Xc int64 [bs,n], Ec int64 [bs,n,n], X_t one-hot, E_t one-hot)."""
    X0, E0, expX, expE = _f32c(X0), _f32c(E0), _f32c(expX), _f32c(expE)
    bs, n, cx = X0.shape
    ce = E0.shape[-1]
    m8 = _mask_u8(node_mask)
    Xc = torch.empty((bs, n), dtype=torch.int64, device=X0.device)
    Ec = torch.empty((bs, n, n), dtype=torch.int64, device=X0.device)
    Xt, Et = torch.empty_like(X0), torch.empty_like(E0)
    _lib.call("mbvae_apply_noise", X0.data_ptr(), E0.data_ptr(), m8.data_ptr(), _f32c(abar_t.reshape(-1)).data_ptr(),
              _f32c(mx).data_ptr(), _f32c(me).data_ptr(), expX.data_ptr(), expE.data_ptr(), Xc.data_ptr(), Ec.data_ptr(),
              Xt.data_ptr(), Et.data_ptr(), bs, n, cx, ce, _stream())
    return Xc, Ec, Xt, Et


@torch.no_grad()
def reverse_sample(logitsX, logitsE, Xt, Et, node_mask, beta_t, abar_s, abar_t, mx, me, expX, expE, want_probs=False):
    """One reverse-diffusion step from denoiser logits.  Returns (Xc, Ec, X_s, E_s[, probX, probE])."""
    logitsX, logitsE, Xt, Et, expX, expE = (_f32c(t) for t in (logitsX, logitsE, Xt, Et, expX, expE))
    bs, n, cx = Xt.shape
    ce = Et.shape[-1]
    m8 = _mask_u8(node_mask)
    dev = Xt.device
    Xc = torch.empty((bs, n), dtype=torch.int64, device=dev)
    Ec = torch.empty((bs, n, n), dtype=torch.int64, device=dev)
    Xs, Es = torch.empty_like(Xt), torch.empty_like(Et)
    pX = torch.empty_like(Xt) if want_probs else None
    pE = torch.empty_like(Et) if want_probs else None
    b, a_s, a_t = (_f32c(t.reshape(-1)) for t in (beta_t, abar_s, abar_t))
    _lib.call("mbvae_reverse_sample", logitsX.data_ptr(), logitsE.data_ptr(), Xt.data_ptr(), Et.data_ptr(), m8.data_ptr(),
              b.data_ptr(), a_s.data_ptr(), a_t.data_ptr(), _f32c(mx).data_ptr(), _f32c(me).data_ptr(), expX.data_ptr(),
              expE.data_ptr(), Xc.data_ptr(), Ec.data_ptr(), Xs.data_ptr(), Es.data_ptr(), _ptr(pX), _ptr(pE), bs, n, cx, ce,
              _stream())
    return (Xc, Ec, Xs, Es, pX, pE) if want_probs else (Xc, Ec, Xs, Es)


# ------------------------------------------------------------------------------------------------ cycle counts
def cycle_counts(A):
    """(per-node 3/4/5-cycle counts [bs,n,3], per-graph 3/4/5/6-cycle counts [bs,4]) of adjacency matrices A [bs,n,n],
    n <= 64 (no gradient: the extra features are inputs of the denoiser)."""
    A = _f32c(A.detach(), "A")
    bs, n = A.shape[0], A.shape[-1]
    xc = torch.empty((bs, n, 3), dtype=torch.float32, device=A.device)
    yc = torch.empty((bs, 4), dtype=torch.float32, device=A.device)
    _lib.call("mbvae_cycle_counts", A.data_ptr(), xc.data_ptr(), yc.data_ptr(), bs, n, _stream())
    return xc, yc
