"""Refusals of the embedding, gated residual norm and gradient clipping operators that the host decides on, without a GPU: the Python
entry points on CPU tensors, and the C entry points on arguments that must never reach a launch."""
import array
import math

import pytest
import torch

from mbvae_amd import _lib, ops

EINVAL, EUNSUPPORTED = -1, -2
A = 0x10000          # stands for a device address: a refused call never looks behind it


def test_python_entry_points_refuse_cpu_tensors():
    w = torch.zeros(5, 8)
    with pytest.raises(RuntimeError, match="no CPU"):
        ops.embedding(torch.zeros(3, dtype=torch.int64), w)
    with pytest.raises(RuntimeError, match="no CPU"):
        ops.gated_residual_norm(torch.zeros(3, 8))
    with pytest.raises(RuntimeError, match="no CPU"):
        ops.clip_grad_norm_([w], 1.0)
    with pytest.raises(RuntimeError, match="no CPU"):
        ops.global_grad_norm([w])


def test_clip_argument_checks():
    g = [torch.zeros(3)]
    with pytest.raises(ValueError, match="outputs"):
        ops.clip_grad_norm_(g, 1.0, out=[])
    for bad in (-1.0, math.nan):
        with pytest.raises(ValueError, match="max_norm"):
            ops.clip_grad_norm_(g, bad)
    for bad in (3.0, 0.5, -math.inf, math.nan):
        with pytest.raises(ValueError, match="norm_type"):
            ops.global_grad_norm(g, bad)
    with pytest.raises(ValueError, match="missing"):
        ops.clip_grad_norm_(g, 1.0, out=[None])


def _clip(src, dst, numel, types, p=2.0, max_norm=1.0, norm=A, ws=A, ws_bytes=None):
    lib = _lib.load()
    n = len(src)
    arrays = [array.array("Q", src), None if dst is None else array.array("Q", dst), array.array("q", numel), array.array("i", types)]
    at = [0 if a is None else a.buffer_info()[0] for a in arrays]
    return lib.mbvae_grad_clip(*at, n, p, max_norm, norm, ws, lib.mbvae_grad_clip_workspace(n) if ws_bytes is None else ws_bytes, 0)


def test_clip_entry_refuses_before_any_launch():
    two = dict(numel=[100, 100], types=[0, 0])
    assert _clip([A, A], [A, A], **two) == EINVAL                       # the same tensor twice, in place
    assert _clip([A, A + 400], [A, A + 396], **two) == EINVAL           # an output over another tensor's last value
    assert _clip([A, A + 4000], [A + 4, A + 4000], **two) == EINVAL     # an output over its own input, shifted
    assert _clip([A, A + 4000], [A + 8000, A + 8200], **two) == EINVAL  # outputs over each other
    assert _clip([A, A + 4000], [A + 4000, A + 8000], **two) == EINVAL  # an output in place of another input
    assert _clip([A + 1], [A + 1], [4], [0]) == EINVAL                  # a float at an odd address
    assert _clip([0], None, [4], [0]) == EINVAL
    assert _clip([A], [0], [4], [0]) == EINVAL
    assert _clip([A], None, [-1], [0]) == EINVAL
    assert _clip([A], None, [4], [3]) == EINVAL
    assert _clip([A], None, [4], [0], p=3.0) == EUNSUPPORTED
    assert _clip([A], [A], [4], [0], max_norm=-1.0) == EINVAL
    assert _clip([A], [A], [4], [0], max_norm=math.nan) == EINVAL
    assert _clip([A], None, [4], [0], norm=0) == EINVAL
    assert _clip([A], None, [4], [0], ws=0) == EINVAL
    assert _clip([A], None, [4], [0], ws=A + 4) == EINVAL
    assert _clip([A], None, [4], [0], ws_bytes=8) == EINVAL


def test_embedding_entries_refuse_before_any_launch():
    lib = _lib.load()

    def fwd(ids=A, id_type=8, w=A, y=A, rows=4, vocab=5, D=8, dtype=0):
        return lib.mbvae_embedding_fwd(ids, id_type, w, y, rows, vocab, D, 1.0, dtype, 0)

    def bwd(ids=A, id_type=8, dy=A, ldy=8, dw=A, rows=4, vocab=5, D=8, dtype=0, ws=A, ws_bytes=1 << 20):
        return lib.mbvae_embedding_bwd(ids, id_type, dy, ldy, dw, rows, vocab, D, 1.0, dtype, ws, ws_bytes, 0)

    for call in (fwd, bwd):
        assert call(rows=-1) == EINVAL and call(vocab=-1) == EINVAL and call(D=-1) == EINVAL
        assert call(id_type=5) == EINVAL and call(dtype=3) == EINVAL and call(ids=0) == EINVAL
        assert call(rows=1 << 31) == EUNSUPPORTED and call(vocab=1 << 31) == EUNSUPPORTED and call(D=(1 << 23) + 1) == EUNSUPPORTED
    assert fwd(w=0) == EINVAL and fwd(y=0) == EINVAL
    assert fwd(rows=0, ids=0, y=0) == 0 and fwd(D=0) == 0
    assert bwd(dy=0) == EINVAL and bwd(dw=0) == EINVAL and bwd(ldy=-1) == EINVAL
    assert bwd(ws=0) == EINVAL and bwd(ws=A + 8) == EINVAL
    assert bwd(ws_bytes=lib.mbvae_embedding_bwd_workspace(4, 5, 8, 0) - 1) == EINVAL
    assert bwd(vocab=0) == 0 and bwd(D=0) == 0


def test_gated_norm_entries_refuse_before_any_launch():
    lib = _lib.load()

    def fwd(x=A, ldx=8, u=A, ldu=8, z=A, ldz=8, pg=A, pb=A, ng=A, nb=A, y=A, n=A, stats=A, rows=4, D=8, eps=1e-5, dtype=0, ptype=0):
        return lib.mbvae_gated_norm_fwd(x, ldx, u, ldu, z, ldz, 0, 1.0, pg, pb, 0, ng, nb, y, n, stats, rows, D, 0, eps, dtype, ptype, 0)

    def bwd(x=A, ldx=8, u=A, ldu=8, z=A, ldz=8, pg=A, pb=A, ng=A, stats=A, dn=A, lddn=8, du=A, dz=A, dpg=A, dng=A, rows=4, D=8, eps=1e-5, dtype=0,
            ptype=0, ws=A, ws_bytes=1 << 20):
        return lib.mbvae_gated_norm_bwd(x, ldx, u, ldu, z, ldz, 0, 1.0, pg, pb, 0, ng, stats, 0, 0, dn, lddn, A, du, dz, 0, dpg, 0, dng, 0, rows, D, 0,
                                        eps, dtype, ptype, ws, ws_bytes, 0)

    for call in (fwd, bwd):
        assert call(x=0) == EINVAL and call(rows=-1) == EINVAL and call(D=0) == EINVAL and call(dtype=3) == EINVAL and call(ptype=-1) == EINVAL
        assert call(ldx=-1) == EINVAL and call(ldu=-1) == EINVAL and call(ldz=-1) == EINVAL and call(eps=-1.0) == EINVAL and call(eps=math.nan) == EINVAL
        assert call(D=8193) == EUNSUPPORTED and call(rows=1 << 31) == EUNSUPPORTED and call(pg=0, pb=A) == EINVAL and call(stats=A + 4) == EINVAL
    assert fwd(y=0) == EINVAL and fwd(n=0) == EINVAL and fwd(ng=0) == EINVAL        # (a beta without its gamma)
    assert fwd(rows=0, x=0) == 0
    assert bwd(ng=0) == EINVAL and bwd(pg=0, pb=0) == EINVAL and bwd(u=0) == EINVAL and bwd(z=0) == EINVAL
    assert bwd(stats=0) == EINVAL and bwd(lddn=-1) == EINVAL and bwd(ws=0) == EINVAL and bwd(ws=A + 8) == EINVAL
    assert bwd(ws_bytes=lib.mbvae_gated_norm_bwd_workspace(4, 8, 0) - 1) == EINVAL


def test_gated_norm_backward_refuses_the_gradient_of_an_absent_vector():
    """Each vector's gradient goes with the vector: nothing is summed for one that is not there, so its place would be filled with whatever the
    workspace holds."""
    lib = _lib.load()

    def bwd(pg=A, scale=A, ng=A, dscale=0, dpg=0, dpb=0, dng=0, dnb=0, rows=4):
        return lib.mbvae_gated_norm_bwd(A, 8, A, 8, A, 8, 0, 1.0, pg, 0, scale, ng, A, A, 8, 0, 8, A, A, A, dscale, dpg, dpb, dng, dnb, rows, 8, 0, 1e-5, 0, 0,
                                        A, 1 << 20, 0)

    for rows in (0, 4):
        assert bwd(scale=0, dscale=A, rows=rows) == EINVAL
        assert bwd(pg=0, dpg=A, rows=rows) == EINVAL and bwd(pg=0, dpb=A, rows=rows) == EINVAL
        assert bwd(ng=0, dng=A, rows=rows) == EINVAL and bwd(ng=0, dnb=A, rows=rows) == EINVAL


def test_denoiser_from_edge_classes_refuses_a_pair_gradient():
    """With the classes at hand the edge input is looked up: E would get the skip connection's gradient and not its whole one."""
    from mbvae_amd.graph_transformer import GraphTransformer
    net = GraphTransformer(n_layers=1, input_dims={"X": 13, "E": 5, "y": 77}, hidden_mlp_dims={"X": 32, "E": 16, "y": 64},
                           hidden_dims={"dx": 64, "de": 16, "dy": 64, "n_head": 4, "dim_ffX": 32, "dim_ffE": 16, "dim_ffy": 64},
                           output_dims={"X": 5, "E": 5, "y": 64})
    E = torch.zeros(2, 3, 3, 5, requires_grad=True)
    args = torch.zeros(2, 3, 13), E, torch.zeros(2, 77), torch.ones(2, 3, dtype=torch.bool)
    ids = torch.zeros(2, 3, 3, dtype=torch.int8)
    with pytest.raises(ValueError, match="gradient of E"):
        net(*args, edge_ids=ids)
    with torch.no_grad(), pytest.raises(RuntimeError):          # (nothing to refuse without gradients: the kernels ask for a GPU next)
        net(*args, edge_ids=ids)


def _clipping_model(grads):
    """A model whose parameters have the given gradients, and an optimiser over them."""
    from mbvae_amd.abstract import AbstractDTIModel
    model = AbstractDTIModel()
    for i, g in enumerate(grads):
        p = torch.nn.Parameter(torch.zeros(g.shape, dtype=g.dtype))
        p.grad = g
        model.register_parameter(f"p{i}", p)
    return model, torch.optim.SGD(model.parameters(), lr=0.1)


def _layouts():
    g = torch.Generator().manual_seed(3)
    a, b = torch.randn(40, 6, generator=g), torch.randn(9, generator=g)
    return {"host": [a, b], "float64": [a.double(), b.double()], "mixed": [a, b.double()], "strided": [a[:, ::2], b],
            "empty": [torch.zeros(0, 3), b], "with history": [a.clone().requires_grad_(True) * 1.0, b]}


@pytest.mark.parametrize("kind", list(_layouts()))
def test_lightning_hook_clips_what_the_kernels_do_not_take(kind):
    """Gradients on the host, in float64, strided or with a history: clipped as Lightning's own hook does, by torch."""
    grads = _layouts()[kind]
    model, opt = _clipping_model(grads)
    want = [t.detach().double().clone() for t in grads]
    norm = math.sqrt(sum(float(t.square().sum()) for t in want))
    model.configure_gradient_clipping(opt, 0.25 * norm)
    for p, t in zip(model.parameters(), want):
        assert torch.allclose(p.grad.detach().double(), 0.25 * t, rtol=1e-5, atol=1e-7)
    assert float(model.logged["train/grad_norm"]) == pytest.approx(norm, rel=1e-5)


def test_lightning_hook_without_anything_to_do():
    """No limit, a limit of zero or below (Lightning clips for neither), and a model without gradients."""
    model, opt = _clipping_model([torch.ones(4)])
    for limit in (None, 0, 0.0, -1.0):
        model.configure_gradient_clipping(opt, limit)
        model.configure_gradient_clipping(opt, limit, "value")
        assert bool((model.p0.grad == 1).all()) and "train/grad_norm" not in model.logged
    model.p0.grad = None
    model.configure_gradient_clipping(opt, 1.0)
    assert float(model.logged["train/grad_norm"]) == 0
