"""Encoders, aggregators and fusion over precomputed feature vectors, on the HIP linear / LayerNorm kernels.

Same constructors, parameter names (state_dict keys) and return values as
mb_vae_dti/training/models/blocks.py (ResidualEncoder :18-66, TransformerEncoder :69-129, ConcatAggregator :136-168,
AttentiveAggregator :171-207, CrossAttentionFusion :214-332).  The module containers (nn.Sequential of
LayerNorm / Linear / activation / Dropout) are kept only to own the parameters under the reference's key names;
forward() walks them and issues the fused kernels.
"""
import torch
import torch.nn as nn
import torch.nn.functional as F

from . import ops


def _ln(ln, x):
    beta = ln.bias if ln.bias is not None else torch.zeros_like(ln.weight)
    return ops.ln_residual(x, None, ln.weight, beta, ln.eps)


def _act_linear(lin, x, activation):
    """activation(lin(x)); ReLU is fused into the GEMM epilogue, other activations run on the (small) output."""
    if isinstance(activation, nn.ReLU):
        return ops.linear(x, lin.weight, lin.bias, act=1)
    return activation(ops.linear(x, lin.weight, lin.bias))


def _lin(lin, x):
    return ops.linear(x, lin.weight, lin.bias)


def _drop(x, p, training):
    return F.dropout(x, p, training) if (training and p > 0) else x


def _mlp_block(seq, x, activation, training):
    """LayerNorm -> Linear -> act -> Dropout -> Linear   (indices 0,1,2,3,4 of the Sequential)."""
    h = _act_linear(seq[1], _ln(seq[0], x), activation)
    return _lin(seq[4], _drop(h, seq[3].p, training))


def _gated(seq, x, u, gate_in, activation, training):
    """x + u * gate(gate_in), gate = LayerNorm -> Linear -> act -> Linear -> Sigmoid -> Dropout (indices 0..5 of the
    Sequential); u None: x + x * gate.  Sigmoid, dropout, product and sum run as one kernel (ops.gate_update)."""
    z = _lin(seq[3], _act_linear(seq[1], _ln(seq[0], gate_in), activation))
    return ops.gate_update(x, u, z, seq[5].p, training)


# ------------------------------------------------------------------------------------------------ fused blocks (ops.set_fused_blocks)
def _affine(ln):
    return ln.weight, ln.bias


def _step(x, u, z, p, training, following):
    """(x + u * dropout(sigmoid(z)), LayerNorm `following` of it) in one kernel; u None: x itself is gated, z None: no gate.  Draws the
    same keep mask as ops.gate_update.  Rows wider than the kernel holds take the separate ones."""
    if x.shape[-1] > ops.GATED_NORM_MAX_WIDTH:
        y = x + u if z is None else ops.gate_update(x, u, z, p, training)
        return y, None if following is None else _ln(following, y)
    keep, scale = None, 1.0
    if z is not None and training and p > 0:
        keep = torch.empty(z.shape, dtype=torch.uint8, device=z.device).bernoulli_(1.0 - p)
        scale = 1.0 / (1.0 - p)
    pre, eps = (None, 1e-5) if following is None else (_affine(following), following.eps)
    return ops.gated_residual_norm(x, u, z, keep=keep, keep_scale=scale, pre=pre, eps=eps)


def _mlp_of(seq, n, activation, training):
    """_mlp_block behind its LayerNorm, whose output n is."""
    return _lin(seq[4], _drop(_act_linear(seq[1], n, activation), seq[3].p, training))


def _gate_of(seq, n, activation):
    """The gate's logits behind its LayerNorm, whose output n is."""
    return _lin(seq[3], _act_linear(seq[1], n, activation))


class ResidualEncoder(nn.Module):
    """Pre-norm residual MLP encoder."""

    def __init__(self, input_dim, hidden_dim, output_dim, n_layers, factor=4, dropout=0.1, bias=True, activation=nn.ReLU()):
        super().__init__()
        self.n_layers, self.activation = n_layers, activation
        self.input_proj = nn.Linear(input_dim, hidden_dim, bias=bias)
        self.layers = nn.ModuleList([
            nn.Sequential(nn.LayerNorm(hidden_dim, bias=bias), nn.Linear(hidden_dim, hidden_dim * factor, bias=bias),
                          self.activation, nn.Dropout(dropout), nn.Linear(hidden_dim * factor, hidden_dim, bias=bias))
            for _ in range(n_layers)])
        self.output_proj = nn.Sequential(nn.LayerNorm(hidden_dim, bias=bias), nn.Linear(hidden_dim, output_dim, bias=bias))

    def forward(self, x):
        x = _lin(self.input_proj, x)
        if ops.fused_blocks():
            norms = [blk[0] for blk in self.layers] + [self.output_proj[0]]
            n = _ln(norms[0], x)
            for blk, following in zip(self.layers, norms[1:]):
                x, n = _step(x, _mlp_of(blk, n, self.activation, self.training), None, 0.0, self.training, following)
            return _lin(self.output_proj[1], n)
        for blk in self.layers:
            x = x + _mlp_block(blk, x, self.activation, self.training)
        return _lin(self.output_proj[1], _ln(self.output_proj[0], x))


class TransformerEncoder(nn.Module):
    """Alternating sigmoid-gate ("attention") and MLP residual blocks on a single feature vector."""

    def __init__(self, input_dim, hidden_dim, output_dim, n_layers, factor=4, dropout=0.1, bias=True, activation=nn.ReLU()):
        super().__init__()
        self.n_layers, self.activation = n_layers, activation
        self.input_proj = nn.Linear(input_dim, hidden_dim, bias=bias)
        self.att_layers, self.mlp_layers = nn.ModuleList(), nn.ModuleList()
        for _ in range(n_layers):
            self.att_layers.append(nn.Sequential(
                nn.LayerNorm(hidden_dim, bias=bias), nn.Linear(hidden_dim, hidden_dim // 4, bias=bias), self.activation,
                nn.Linear(hidden_dim // 4, hidden_dim, bias=bias), nn.Sigmoid(), nn.Dropout(dropout)))
            self.mlp_layers.append(nn.Sequential(
                nn.LayerNorm(hidden_dim, bias=bias), nn.Linear(hidden_dim, hidden_dim * factor, bias=bias), self.activation,
                nn.Dropout(dropout), nn.Linear(hidden_dim * factor, hidden_dim, bias=bias)))
        self.output_proj = nn.Sequential(nn.LayerNorm(hidden_dim, bias=bias), nn.Linear(hidden_dim, output_dim, bias=bias))

    def forward(self, x):
        x = _lin(self.input_proj, x)
        if ops.fused_blocks():
            act, tr = self.activation, self.training
            norms = [att[0] for att in self.att_layers] + [self.output_proj[0]]
            n = _ln(norms[0], x)
            for att, mlp, following in zip(self.att_layers, self.mlp_layers, norms[1:]):
                x, n = _step(x, None, _gate_of(att, n, act), att[5].p, tr, mlp[0])
                x, n = _step(x, _mlp_of(mlp, n, act, tr), None, 0.0, tr, following)
            return _lin(self.output_proj[1], n)
        for att, mlp in zip(self.att_layers, self.mlp_layers):
            x = _gated(att, x, None, x, self.activation, self.training)
            x = x + _mlp_block(mlp, x, self.activation, self.training)
        return _lin(self.output_proj[1], _ln(self.output_proj[0], x))


class ConcatAggregator(nn.Module):
    def __init__(self, input_dim, output_dim, n_features, dropout=0.1, activation=nn.ReLU()):
        super().__init__()
        self.activation = activation
        total = input_dim * n_features
        self.projection = nn.Sequential(nn.LayerNorm(total), nn.Linear(total, output_dim), self.activation, nn.Dropout(dropout))

    def forward(self, features):
        h = _act_linear(self.projection[1], _ln(self.projection[0], torch.cat(features, dim=-1)), self.activation)
        return _drop(h, self.projection[3].p, self.training)


class AttentiveAggregator(nn.Module):
    """Softmax-weighted sum over the views (weights from a 1x1 conv), then LayerNorm-Linear-act-Dropout."""

    def __init__(self, input_dim, output_dim, n_features, dropout=0.1, activation=nn.ReLU()):
        super().__init__()
        self.activation = activation
        self.to_attn_logits = nn.Conv1d(input_dim, 1, 1)
        self.projection = nn.Sequential(nn.LayerNorm(input_dim), nn.Linear(input_dim, output_dim), self.activation, nn.Dropout(dropout))

    def forward(self, features):
        # Views in the middle and the logits as one product: torch would sum over the columns of [B, D, V], and over all rows for the
        # logits' weight, with several blocks an output, whose counters it clears by a memory-set node in a captured graph.
        stacked = torch.stack(features, dim=1)                                         # [B, V, D]
        rows = stacked.reshape(-1, stacked.shape[-1])
        logits = ops.linear(rows, self.to_attn_logits.weight.reshape(1, -1), self.to_attn_logits.bias).reshape(stacked.shape[:2])
        attn = F.softmax(logits, dim=-1).unsqueeze(1)                                  # [B, 1, V]
        agg = (stacked * attn.transpose(1, 2)).sum(dim=1)
        h = _act_linear(self.projection[1], _ln(self.projection[0], agg), self.activation)
        return _drop(h, self.projection[3].p, self.training), attn


class CrossAttentionFusion(nn.Module):
    """n_layers x (bidirectional gated cross update, self gate, MLP) on the drug / target pair, then attentive
    aggregation; returns (fused, attention weights)."""

    def __init__(self, input_dim, output_dim, n_layers, factor=4, dropout=0.1, bias=True, activation=nn.ReLU()):
        super().__init__()
        self.n_layers, self.activation = n_layers, activation
        names = ("cross_gates_a_to_b", "cross_gates_b_to_a", "align_proj_b_to_a", "align_proj_a_to_b", "self_gates_a",
                 "self_gates_b", "mlp_a", "mlp_b")
        for nm in names:
            setattr(self, nm, nn.ModuleList())

        def gate(width):
            return nn.Sequential(nn.LayerNorm(width, bias=bias), nn.Linear(width, input_dim // factor, bias=bias), self.activation,
                                 nn.Linear(input_dim // factor, input_dim, bias=bias), nn.Sigmoid(), nn.Dropout(dropout))

        def mlp():
            return nn.Sequential(nn.LayerNorm(input_dim, bias=bias), nn.Linear(input_dim, input_dim // factor, bias=bias),
                                 self.activation, nn.Dropout(dropout), nn.Linear(input_dim // factor, input_dim, bias=bias))

        for _ in range(n_layers):
            self.align_proj_b_to_a.append(nn.Linear(input_dim, input_dim, bias=False))
            self.align_proj_a_to_b.append(nn.Linear(input_dim, input_dim, bias=False))
            self.cross_gates_a_to_b.append(gate(input_dim * 2))
            self.cross_gates_b_to_a.append(gate(input_dim * 2))
            self.self_gates_a.append(gate(input_dim))
            self.self_gates_b.append(gate(input_dim))
            self.mlp_a.append(mlp())
            self.mlp_b.append(mlp())
        self.att_agg = AttentiveAggregator(input_dim=input_dim, output_dim=output_dim, n_features=2, dropout=dropout,
                                           activation=activation)

    def forward(self, a, b):
        act, tr = self.activation, self.training
        for i in range(self.n_layers if ops.fused_blocks() else 0):
            gate_a, gate_b, self_a, self_b = self.cross_gates_b_to_a[i], self.cross_gates_a_to_b[i], self.self_gates_a[i], self.self_gates_b[i]
            ab, ba = torch.cat([a, b], dim=-1), torch.cat([b, a], dim=-1)
            ua, ub = _lin(self.align_proj_b_to_a[i], b), _lin(self.align_proj_a_to_b[i], a)
            a, na = _step(a, ua, _gate_of(gate_a, _ln(gate_a[0], ab), act), gate_a[5].p, tr, self_a[0])
            b, nb = _step(b, ub, _gate_of(gate_b, _ln(gate_b[0], ba), act), gate_b[5].p, tr, self_b[0])
            a, na = _step(a, None, _gate_of(self_a, na, act), self_a[5].p, tr, self.mlp_a[i][0])
            b, nb = _step(b, None, _gate_of(self_b, nb, act), self_b[5].p, tr, self.mlp_b[i][0])
            a = a + _mlp_of(self.mlp_a[i], na, act, tr)
            b = b + _mlp_of(self.mlp_b[i], nb, act, tr)
        for i in range(0 if ops.fused_blocks() else self.n_layers):
            a, b = (_gated(self.cross_gates_b_to_a[i], a, _lin(self.align_proj_b_to_a[i], b), torch.cat([a, b], dim=-1), act, tr),
                    _gated(self.cross_gates_a_to_b[i], b, _lin(self.align_proj_a_to_b[i], a), torch.cat([b, a], dim=-1), act, tr))
            a = _gated(self.self_gates_a[i], a, None, a, act, tr)
            b = _gated(self.self_gates_b[i], b, None, b, act, tr)
            a = a + _mlp_block(self.mlp_a[i], a, act, tr)
            b = b + _mlp_block(self.mlp_b[i], b, act, tr)
        return self.att_agg([a, b])
