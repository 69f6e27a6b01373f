"""Embedding, gated residual norm and gradient clipping on the GPU against 64-bit references (tests/_train_operators.py holds the formulas and
the derivation of every bound)."""
import math

import pytest
import torch

from tests._train_operators import (U, check, clip_reference, embedding_gradient, embedding_reference, gated_reference, half_step, tiny)

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.fixture()
def ops():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from mbvae_amd import ops as module
    return module


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _randn(g, *shape, dtype=F32):
    return torch.randn(*shape, generator=g).to(dtype)


# ------------------------------------------------------------------------------------------------ embedding
def _ids(g, rows, V, kind, dtype, pad=0.1):
    u = torch.rand(rows, generator=g)
    if kind == "uniform":
        ids = (u * V).long().clamp(max=max(V - 1, 0))
    elif kind == "hot":                        # nine tenths of all tokens are one id
        ids = torch.where(u < 0.9, V // 2, (torch.rand(rows, generator=g) * V).long().clamp(max=max(V - 1, 0)))
    elif kind == "sorted":
        ids = (u.sort().values * V).long().clamp(max=max(V - 1, 0))
    elif kind == "one":
        return torch.full((rows,), V - 1).to(dtype)
    else:                                      # no id of the table at all
        ids = torch.where(u < 0.5, -1, V if V <= torch.iinfo(dtype).max else -1)
        return ids.to(dtype)
    return torch.where(torch.rand(rows, generator=g) < pad, -1, ids).to(dtype)


EMBEDDING = [
    # rows, V, D, table type, id type, spread of the ids
    (1, 1, 1, F32, torch.int64, "uniform"), (1, 5, 64, BF16, torch.int8, "uniform"), (3, 2, 7, F16, torch.int16, "none"),
    (64, 5, 256, F32, torch.int8, "uniform"), (65, 127, 33, F32, torch.int8, "hot"), (1000, 128, 5, BF16, torch.int32, "uniform"),
    (257, 255, 130, F16, torch.int32, "uniform"), (257, 256, 64, F32, torch.int32, "uniform"), (300, 257, 65, F32, torch.int16, "sorted"),
    (8191, 700, 12, F32, torch.int64, "hot"), (8192, 70000, 9, F32, torch.int32, "uniform"), (8193, 300, 24, BF16, torch.int64, "uniform"),
    (20000, 5, 64, F32, torch.int8, "hot"), (20000, 4170, 48, F16, torch.int32, "sorted"), (40000, 3, 16, F32, torch.int8, "one"),
    (70001, 66000, 20, F32, torch.int64, "hot"), (30000, 9, 1037, BF16, torch.int8, "uniform"), (16385, 11, 8, F32, torch.int8, "none"),
    (17, 20, 2050, F32, torch.int64, "uniform"), (700, 32, 260, F32, torch.int8, "hot"), (700, 33, 260, F32, torch.int8, "hot"), (3000, 16, 520, BF16, torch.int16, "uniform"),
    (3000, 17, 520, BF16, torch.uint8, "hot"), (32768, 4000, 16, F32, torch.int64, "hot"), (32769, 4000, 16, F32, torch.int64, "hot"), (32768, 33, 8, F16, torch.int8, "one"),
    (900, 65535, 8, F32, torch.int32, "uniform"), (900, 65536, 8, F32, torch.int64, "uniform"),
    (5000, 128000, 8, F32, torch.int64, "uniform"), (9000, 262143, 4, BF16, torch.int32, "hot"), (900, 262144, 4, F32, torch.int64, "sorted"), (33000, 128000, 4, F16, torch.int64, "hot"), (2, 65000, 4, BF16, torch.int64, "uniform"), (5000, 1, 40, F32, torch.int64, "uniform"),
]


@pytest.mark.parametrize("rows,V,D,dtype,id_dtype,kind", EMBEDDING)
def test_embedding_forward_and_gradient(ops, rows, V, D, dtype, id_dtype, kind):
    g = _gen(rows + V + D)
    ids = _ids(g, rows, V, kind, id_dtype)
    w, dy = _randn(g, V, D, dtype=dtype), _randn(g, rows, D, dtype=dtype)
    scale = D ** 0.5
    want, bound = embedding_reference(ids, w, scale)
    weight = w.cuda().requires_grad_(True)
    y = ops.embedding(ids.cuda(), weight, scale)
    assert y.dtype == dtype
    check(y, want, bound, "y")
    with torch.no_grad():
        assert torch.equal(ops.embedding(ids.cuda(), weight, scale), y.detach())
    dw, = torch.autograd.grad(y, weight, dy.cuda())
    want, bound = embedding_gradient(ids, dy, V, scale)
    assert dw.dtype == dtype
    check(dw, want, bound, "dweight")
    y = ops.embedding(ids.cuda(), weight, scale)
    again, = torch.autograd.grad(y, weight, dy.cuda())
    assert torch.equal(again, dw), "the same call gives other bits"


@pytest.mark.parametrize("lengths", [[16], [16, 16], [32, 16], [15, 17, 16], [33, 1, 14], [1, 15, 16, 48], [47, 17], [31, 1, 1, 31], [5, 16, 11, 16, 16], [64, 1],
                                     [8, 40, 16], [17, 47, 1, 16], [16, 17, 15, 1, 33, 14, 80, 3], [160, 160, 7], [1] * 50, [2, 30] * 8, [129, 255, 1, 127]])
@pytest.mark.parametrize("many", [False, True])
def test_embedding_gradient_runs_meet_chunks(ops, lengths, many):
    """Runs of equal ids that begin and end on, before and behind multiples of 16 tokens, at the end of the tokens and before padding; with
    `many` behind 33 000 tokens of smaller ids, which take the radix sort and another chunk length."""
    g = _gen(len(lengths) + sum(lengths))
    V, D = 1000, 24
    ids = torch.cat([torch.full((n,), 40 + 3 * k) for k, n in enumerate(lengths)])
    if many:
        ids = torch.cat((torch.arange(33 * 1024) % 33, ids))
    for pad in (0, 1, 16, 21):
        every = torch.cat((ids, torch.full((pad,), -1)))
        every = every[torch.randperm(every.numel(), generator=g)]
        dy = _randn(g, every.numel(), D)
        weight = _randn(g, V, D).cuda().requires_grad_(True)
        dw, = torch.autograd.grad(ops.embedding(every.cuda(), weight, 0.5), weight, dy.cuda())
        want, bound = embedding_gradient(every, dy, V, 0.5)
        check(dw, want, bound, f"dweight, {pad} rows of padding")


def test_embedding_shapes_strides_and_ids_outside(ops):
    g = _gen(1)
    w = _randn(g, 6, 20)
    ids = torch.tensor([[0, 5, -1, 6], [3, -128, 127, 2]], dtype=torch.int8)
    want, bound = embedding_reference(ids.reshape(-1), w, 2.0)
    got = ops.embedding(ids.cuda(), w.cuda(), 2.0)
    assert got.shape == (2, 4, 20)
    check(got.reshape(8, 20), want, bound, "y")
    assert not bool(got[0, 2:].any()) and not bool(got[1, 1:3].any())
    # ids and table of other layouts, a gradient with strided rows and an expanded one
    table = w.t().contiguous().cuda().t().requires_grad_(True)
    strided = ids.t().contiguous().cuda().t()
    y = ops.embedding(strided, table, 2.0)
    assert torch.equal(y, got)
    wide = _randn(g, 2, 4, 40)
    for dy in (wide.cuda()[..., 3:23], torch.ones(1, 1, 1).cuda().expand(2, 4, 20), wide.cuda()[..., ::2]):
        dw, = torch.autograd.grad(ops.embedding(strided, table, 2.0), table, dy)
        want, bound = embedding_gradient(ids, dy.contiguous(), 6, 2.0)
        check(dw, want, bound, "dweight")
    # the largest ids of each type, and values that only fit 64 bits
    far = torch.tensor([2 ** 40, -2 ** 40, 2 ** 32, 2 ** 32 + 1, 1], dtype=torch.int64).cuda()
    got = ops.embedding(far, table.detach(), 1.0)
    assert not bool(got[:4].any()) and torch.equal(got[4].cpu(), w[1])
    byte = torch.tensor([255, 0, 5], dtype=torch.uint8).cuda()
    assert not bool(ops.embedding(byte, table.detach()).cpu()[0].any())


def test_embedding_of_nothing(ops):
    w = torch.randn(5, 8, device="cuda", requires_grad=True)
    none = torch.zeros(0, dtype=torch.int64, device="cuda")
    y = ops.embedding(none, w)
    assert y.shape == (0, 8)
    dw, = torch.autograd.grad(y, w, torch.zeros_like(y))
    assert dw.shape == w.shape and not bool(dw.any())
    empty = torch.zeros(0, 8, device="cuda", requires_grad=True)
    y = ops.embedding(torch.tensor([0, -1, 3], device="cuda"), empty)
    assert y.shape == (3, 8) and not bool(y.any())
    assert torch.autograd.grad(y, empty, torch.ones_like(y))[0].shape == (0, 8)
    thin = torch.zeros(4, 0, device="cuda", requires_grad=True)
    y = ops.embedding(none, thin)
    assert y.shape == (0, 0) and torch.autograd.grad(y, thin, y)[0].shape == (4, 0)


def test_embedding_keeps_non_finite_rows_apart(ops):
    """A row of the gradient that is not finite reaches its own row of the table and no other; padding rows reach none."""
    ids = torch.tensor([0, 1, -1, 2, 1, -1] * 50, dtype=torch.int8)
    dy = torch.ones(300, 12)
    dy[2::6] = math.nan
    dy[5::6] = math.inf
    dy[1] = math.inf
    w = torch.full((4, 12), 2.0)
    w[3] = math.nan
    weight = w.cuda().requires_grad_(True)
    y = ops.embedding(ids.cuda(), weight, math.inf)
    assert bool(torch.isinf(y[0]).all()) and not bool(y[2].any()), "padding stays zero whatever the scale"
    y = ops.embedding(ids.cuda(), weight)
    assert bool(torch.isfinite(y).all())
    dw = torch.autograd.grad(y, weight, dy.cuda())[0].cpu()
    assert torch.equal(dw[0], torch.full((12,), 50.0)) and torch.equal(dw[2], torch.full((12,), 50.0))
    assert bool(torch.isinf(dw[1]).all()) and not bool(dw[3].any())


def test_embedding_gradient_against_differences(ops):
    g = _gen(4)
    ids, w, dy = torch.randint(-1, 7, (40,), generator=g), _randn(g, 7, 6), _randn(g, 40, 6)
    weight = w.cuda().requires_grad_(True)
    dw, = torch.autograd.grad(ops.embedding(ids.cuda(), weight, 1.5), weight, dy.cuda())
    step, direction = 0.25, _randn(g, 7, 6)
    up, down = (float((ops.embedding(ids.cuda(), (w + s * step * direction).cuda(), 1.5).double().cpu() * dy).sum()) for s in (1, -1))
    # the function is linear: only the rounding of the two values (240 products each) separates the difference from the gradient
    size = float((embedding_reference(ids, w.abs() + direction.abs(), 1.5)[0] * dy.abs()).sum())
    assert abs((up - down) / (2 * step) - float((dw.double().cpu() * direction).sum())) <= size * 16 * U / step


def test_embedding_refusals(ops):
    w = torch.zeros(5, 8, device="cuda")
    with pytest.raises(RuntimeError, match="integer ids"):
        ops.embedding(torch.zeros(3, device="cuda"), w)
    with pytest.raises(RuntimeError, match="integer ids"):
        ops.embedding(torch.zeros(3, dtype=torch.int64), w)
    with pytest.raises(RuntimeError, match="float32"):
        ops.embedding(torch.zeros(3, dtype=torch.int64, device="cuda"), w.double())
    with pytest.raises(ValueError, match=r"\[V, D\]"):
        ops.embedding(torch.zeros(3, dtype=torch.int64, device="cuda"), w[0])
    with pytest.raises(RuntimeError):
        y = ops.embedding(torch.zeros(3, dtype=torch.int64, device="cuda"), w.requires_grad_(True))
        dw, = torch.autograd.grad(y.sum(), w, create_graph=True)
        torch.autograd.grad(dw.sum(), w)


# ------------------------------------------------------------------------------------------------ gated residual norm
def _block(g, shape, dtype, ptype, own_u, gate, keep, post, scale, pre, norm, betas=True):
    D = shape[-1]

    def affine():
        return (1 + 0.2 * _randn(g, D)).to(ptype), (0.3 * _randn(g, D)).to(ptype) if betas else None

    return dict(x=_randn(g, *shape, dtype=dtype), u=_randn(g, *shape, dtype=dtype) if own_u else None, z=(2 * _randn(g, *shape)).to(dtype) if gate else None,
                keep=(torch.rand(shape, generator=g) < 0.8).to(torch.uint8) if keep else None, keep_scale=1.25 if keep else 1.0,
                post=affine() if post else None, scale=(0.6 * _randn(g, D)).to(ptype) if scale else None, pre=affine() if pre else None, norm=norm)


def _device(t, grad=True):
    if t is None:
        return None
    if isinstance(t, tuple):
        return tuple(_device(v, grad) for v in t)
    return t.cuda().requires_grad_(grad) if t.is_floating_point() else t.cuda()


def _leaves(b):
    every = {"x": b["x"], "u": b["u"], "z": b["z"], "scale": b["scale"]}
    for side in ("post", "pre"):
        if b[side] is not None:
            every[side + "_gamma"], every[side + "_beta"] = b[side]
    return {k: t for k, t in every.items() if t is not None}


def _call(ops, b, eps):
    return ops.gated_residual_norm(b["x"], b["u"], b["z"], keep=b["keep"], keep_scale=b["keep_scale"], post=b["post"], res_scale=b["scale"], pre=b["pre"],
                                   norm=b["norm"], eps=eps)


def _run_block(ops, host, dy, dn, eps=1e-5, dev=None):
    b = dev or {k: _device(v) if k not in ("keep_scale", "norm") else v for k, v in host.items()}
    y, n = _call(ops, b, eps)
    leaves = _leaves(b)
    pairs = [(o, d.cuda()) for o, d in ((y, dy), (n, dn)) if o is not None and d is not None]
    grads = torch.autograd.grad([o for o, _ in pairs], list(leaves.values()), [d for _, d in pairs])
    want = gated_reference(**host, eps=eps, dy=dy, dn=dn if n is not None else None)
    got = {"y": y, "n": n, **{"d" + k: t for k, t in zip(leaves, grads)}}
    for k, (value, bound) in want.items():
        assert got[k].dtype == (host["x"].dtype if k in ("y", "n", "dx", "du", "dz") else leaves[k[1:]].dtype), k
        check(got[k], value, bound, k)
    assert set(want) == {k for k, v in got.items() if v is not None}
    return got


BLOCK = [
    # shape, type, parameters' type, u, gate, keep, post, scale, pre, norm
    ((1, 1), F32, F32, True, True, False, True, True, True, "layer"), ((1, 512), F32, F32, False, True, False, False, False, True, "layer"),
    ((3, 2), F32, F32, True, False, False, True, True, True, "rms"), ((256, 512), F32, F32, False, True, True, False, False, True, "layer"),
    ((33, 64), F32, F32, True, True, False, False, False, True, "layer"), ((1000, 64), BF16, BF16, True, True, True, True, True, True, "layer"),
    ((70, 77), F16, F32, True, True, False, True, True, True, "rms"), ((129, 130), F32, F32, True, True, True, True, True, True, "layer"),
    ((65, 256), BF16, F32, True, True, False, True, True, True, "layer"), ((31, 257), F32, F32, True, False, False, True, False, True, "rms"),
    ((19, 513), F16, F16, True, True, True, True, True, True, "layer"), ((9, 1024), F32, F32, True, True, False, True, True, True, "rms"),
    ((50, 1037), F16, F32, True, False, False, True, True, True, "rms"), ((7, 2048), BF16, F32, True, True, True, True, True, True, "layer"),
    ((5, 2049), F32, F32, True, True, False, True, True, True, "layer"), ((4, 4096), BF16, BF16, False, True, True, True, True, True, "rms"),
    ((3, 4100), F32, F32, True, True, True, True, True, True, "layer"), ((2, 8192), F16, F32, True, True, False, True, True, True, "layer"),
    ((9, 8191), F32, F32, False, False, False, True, True, True, "rms"), ((2, 3, 5, 40), F32, F32, True, True, True, True, True, True, "layer"),
    ((20, 100), F32, F32, True, True, True, True, True, False, "layer"), ((20, 100), BF16, F32, True, True, False, False, True, False, "rms"),
    ((20, 96), F32, F32, False, False, True, False, False, False, "layer"), ((5000, 128), F32, F32, True, True, False, True, True, True, "layer"),
    ((20, 96), F32, F32, True, False, False, False, False, True, "layer"), ((4097, 16), BF16, F32, True, True, False, True, True, True, "rms"),
]


@pytest.mark.parametrize("shape,dtype,ptype,own_u,gate,keep,post,scale,pre,norm", BLOCK)
def test_gated_residual_norm(ops, shape, dtype, ptype, own_u, gate, keep, post, scale, pre, norm):
    g = _gen(sum(shape) + 7 * own_u + gate)
    host = _block(g, shape, dtype, ptype, own_u, gate, keep, post, scale, pre, norm, betas=norm == "layer")
    dy, dn = _randn(g, *shape, dtype=dtype), _randn(g, *shape, dtype=dtype)
    first = _run_block(ops, host, dy, dn)
    again = _run_block(ops, host, dy, dn)
    for k in first:
        assert first[k] is None or torch.equal(first[k], again[k]), f"{k}: the same call gives other bits"
    with torch.no_grad():
        y, n = _call(ops, {k: _device(v, False) if k not in ("keep_scale", "norm") else v for k, v in host.items()}, 1e-5)
    assert torch.equal(y, first["y"]) and (n is None or torch.equal(n, first["n"]))


@pytest.mark.parametrize("side", ["y", "n"])
def test_gated_residual_norm_one_output_used(ops, side):
    g = _gen(8)
    host = _block(g, (37, 72), F32, F32, True, True, True, True, True, True, "layer")
    d = _randn(g, 37, 72)
    b = {k: _device(v) if k not in ("keep_scale", "norm") else v for k, v in host.items()}
    y, n = _call(ops, b, 1e-5)
    leaves = _leaves(b)
    grads = torch.autograd.grad(y if side == "y" else n, list(leaves.values()), d.cuda(), allow_unused=True)
    want = gated_reference(**host, eps=1e-5, dy=d if side == "y" else None, dn=d if side == "n" else None)
    for k, t in zip(leaves, grads):
        if "d" + k in want:
            check(t, *want["d" + k], "d" + k)
        else:
            assert t is None or not bool(t.any()), k


def test_gated_residual_norm_some_leaves_frozen(ops):
    """Only what asks for a gradient gets one, and it is the one of the full call."""
    g = _gen(9)
    host = _block(g, (21, 65), F32, F32, True, True, True, True, True, True, "layer")
    dy, dn = _randn(g, 21, 65), _randn(g, 21, 65)
    full = _run_block(ops, host, dy, dn)
    names = list(_leaves({k: _device(v) if k not in ("keep_scale", "norm") else v for k, v in host.items()}))
    for wanted in (["x"], ["u"], ["z"], ["scale", "pre_beta"], ["post_gamma"], ["post_beta", "x"], ["pre_gamma", "z"]):
        b = {k: _device(v, False) if k not in ("keep_scale", "norm") else v for k, v in host.items()}
        leaves = _leaves(b)
        for k in wanted:
            leaves[k].requires_grad_(True)
        y, n = _call(ops, b, 1e-5)
        grads = torch.autograd.grad([y, n], [leaves[k] for k in wanted], [dy.cuda(), dn.cuda()])
        for k, t in zip(wanted, grads):
            assert torch.equal(t, full["d" + k]), k
    assert "post_beta" in names


def test_gated_residual_norm_strided_operands(ops):
    """Halves of one projection's output, rows further apart than they are long, expanded and transposed operands and gradients."""
    g = _gen(10)
    for D, dtype in ((64, F32), (77, BF16), (1037, F16), (300, F32)):
        R = 23
        both, wide, dd = _randn(g, R, 2 * D, dtype=dtype), _randn(g, R, D + 5, dtype=dtype), _randn(g, R, 3 * D, dtype=dtype)
        u, z = both.chunk(2, -1)
        host = _block(g, (R, D), dtype, F32, True, True, False, True, True, True, "layer")
        host.update(x=wide[:, 3:3 + D], u=u, z=z)
        dev = {k: _device(v) if k not in ("keep_scale", "norm") else v for k, v in host.items()}
        du, dz = both.cuda().chunk(2, -1)
        dev.update(x=wide.cuda()[:, 3:3 + D].requires_grad_(True), u=du.detach().requires_grad_(True), z=dz.detach().requires_grad_(True))
        y, n = _call(ops, dev, 1e-5)
        leaves = _leaves(dev)
        for dy, dn in ((dd[:, :D], dd[:, D + 1:2 * D + 1]), (dd[:1, :D].expand(R, D), dd[:, 2 * D:]), (dd[:, :1].expand(R, D), dd.view(3 * D, R)[:D].t())):
            gy = dd.cuda()
            gy, gn = {0: (gy[:, :D], gy[:, D + 1:2 * D + 1]), 1: (gy[:1, :D].expand(R, D), gy[:, 2 * D:]),
                      2: (gy[:, :1].expand(R, D), gy.view(3 * D, R)[:D].t())}[0 if dy.stride(0) > 1 and dy.stride(1) == 1 else 1 if dy.stride(0) == 0 else 2]
            grads = torch.autograd.grad([y, n], list(leaves.values()), [gy, gn], retain_graph=True)
            want = gated_reference(**{**host, "x": host["x"].contiguous()}, eps=1e-5, dy=dy.contiguous(), dn=dn.contiguous())
            check(y, *want["y"], "y")
            check(n, *want["n"], "n")
            for k, t in zip(leaves, grads):
                check(t, *want["d" + k], f"d{k} D={D}")
    row = _randn(g, 1, 96)
    host = _block(g, (11, 96), F32, F32, True, True, False, False, False, True, "layer")
    host["x"] = row.expand(11, 96)
    leaf = row.cuda().requires_grad_(True)
    dev = {k: _device(v) if k not in ("keep_scale", "norm") else v for k, v in host.items()}
    dev["x"] = leaf.expand(11, 96)
    y, n = _call(ops, dev, 1e-5)
    want = gated_reference(**host, eps=1e-5, dy=torch.ones(11, 96), dn=torch.ones(11, 96))
    check(y, *want["y"], "y of a broadcast x")
    dx, = torch.autograd.grad([y, n], [leaf], [torch.ones_like(y), torch.ones_like(n)])
    value, bound = want["dx"]
    check(dx, value.sum(0, keepdim=True), bound.sum(0, keepdim=True) + 11 * U * value.abs().sum(0, keepdim=True), "gradient of a broadcast x")


def test_gated_residual_norm_dropped_and_non_finite_values(ops):
    """A dropped value adds nothing and takes no gradient, whatever u and z hold there; a row that drops everything passes x on."""
    g = _gen(11)
    R, D = 24, 80
    host = _block(g, (R, D), F32, F32, True, True, True, False, True, True, "layer")
    keep = host["keep"]
    keep[0] = 0
    u, z = host["u"].clone(), host["z"].clone()
    u[keep == 0] = math.nan
    z[keep == 0] = math.inf
    z[1], z[2] = 200.0, -200.0                     # a gate that is open or shut to the last bit
    z[1][keep[1] == 0] = -math.inf
    clean = {**host, "u": torch.where(keep == 0, 0.0, u), "z": torch.where(keep == 0, 0.0, z)}
    dy, dn = _randn(g, R, D), _randn(g, R, D)
    dev = {k: _device(v) if k not in ("keep_scale", "norm") else v for k, v in {**host, "u": u, "z": z}.items()}
    y, n = _call(ops, dev, 1e-5)
    leaves = _leaves(dev)
    grads = dict(zip(leaves, torch.autograd.grad([y, n], list(leaves.values()), [dy.cuda(), dn.cuda()])))
    want = gated_reference(**clean, eps=1e-5, dy=dy, dn=dn)
    check(y, *want["y"], "y")
    check(n, *want["n"], "n")
    for k, t in grads.items():
        check(t, *want["d" + k], "d" + k)
    assert torch.equal(y[0].cpu(), host["x"][0]) and not bool(grads["u"][0].any()) and not bool(grads["z"][0].any())
    # a row that is not finite stays in its row
    u = host["u"].clone()
    u[5] = math.nan
    host2 = {**host, "u": u, "keep": None, "keep_scale": 1.0, "post": host["pre"]}
    y, n = _call(ops, {k: _device(v, False) if k not in ("keep_scale", "norm") else v for k, v in host2.items()}, 1e-5)
    bad = torch.isnan(n).any(1).cpu()
    assert bool(bad[5]) and int(bad.sum()) == 1


def test_gated_residual_norm_rows_without_spread(ops):
    """Rows of one value (LayerNorm's deviation is eps alone) and rows far from zero."""
    g = _gen(12)
    for norm in ("layer", "rms"):
        host = _block(g, (12, 96), F32, F32, True, False, False, True, False, True, norm)
        host["x"][0], host["u"][0] = 3.0, 0.5
        host["x"][1], host["u"][1] = 0.0, 0.0
        host["x"][2] = 1000 + host["x"][2]
        _run_block(ops, host, _randn(g, 12, 96), _randn(g, 12, 96))


def test_gated_residual_norm_of_nothing(ops):
    x = torch.zeros(0, 40, device="cuda", requires_grad=True)
    gamma, beta = torch.ones(40, device="cuda", requires_grad=True), torch.zeros(40, device="cuda", requires_grad=True)
    y, n = ops.gated_residual_norm(x, x, x, post=(gamma, beta), pre=(gamma, beta))
    assert y.shape == n.shape == (0, 40)
    dx, dg, db = torch.autograd.grad([y, n], [x, gamma, beta], [y.detach(), n.detach()])
    assert dx.shape == (0, 40) and not bool(dg.any()) and not bool(db.any())
    y, n = ops.gated_residual_norm(torch.zeros(2, 0, 40, device="cuda"))
    assert y.shape == (2, 0, 40) and n is None


def test_gated_residual_norm_gradient_against_differences(ops):
    """Central differences of the operator's own forward along one direction, all leaves at once.  The difference's own error: third
    derivatives times step^2 / 6 against the rounding of two sums over step; a step of 1e-2 leaves both below 1e-3 of the sum of magnitudes."""
    g = _gen(13)
    host = _block(g, (6, 48), F32, F32, True, True, True, True, True, True, "layer")
    dy, dn = _randn(g, 6, 48), _randn(g, 6, 48)
    dev = {k: _device(v) if k not in ("keep_scale", "norm") else v for k, v in host.items()}
    leaves = _leaves(dev)
    y, n = _call(ops, dev, 1e-5)
    grads = torch.autograd.grad([y, n], list(leaves.values()), [dy.cuda(), dn.cuda()])
    ways = {k: _randn(g, *t.shape).cuda() for k, t in leaves.items()}
    slope = sum(float((d.double() * ways[k].double()).sum()) for d, k in zip(grads, leaves))
    size = sum(float((d.double() * ways[k].double()).abs().sum()) for d, k in zip(grads, leaves))
    step, values = 1e-2, []
    with torch.no_grad():
        for s in (step, -step):
            moved = {k: t + s * ways[k] for k, t in leaves.items()}
            b = {**dev, "x": moved["x"], "u": moved["u"], "z": moved["z"], "scale": moved["scale"], "post": (moved["post_gamma"], moved["post_beta"]),
                 "pre": (moved["pre_gamma"], moved["pre_beta"])}
            y, n = _call(ops, b, 1e-5)
            values.append(float((y.double() * dy.cuda()).sum() + (n.double() * dn.cuda()).sum()))
    assert abs((values[0] - values[1]) / (2 * step) - slope) <= 1e-3 * size


def test_gated_residual_norm_cannot_be_differentiated_twice(ops):
    g = _gen(14)
    host = _block(g, (5, 24), F32, F32, True, True, False, True, True, True, "layer")
    dev = {k: _device(v) if k not in ("keep_scale", "norm") else v for k, v in host.items()}
    leaves = _leaves(dev)
    y, n = _call(ops, dev, 1e-5)
    once = torch.autograd.grad((y * n).sum(), list(leaves.values()), retain_graph=True)
    graph = torch.autograd.grad((y * n).sum(), list(leaves.values()), create_graph=True)
    for a, b in zip(once, graph):
        assert torch.equal(a, b)
    with pytest.raises(RuntimeError, match="twice"):
        graph[0].sum().backward(retain_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(graph[0].sum(), leaves["x"])


def test_gated_residual_norm_refusals(ops):
    x = torch.zeros(4, 16, device="cuda")
    ones = torch.ones(16, device="cuda")
    for kwargs, match in ((dict(u=torch.zeros(4, 8, device="cuda")), "shape"), (dict(u=x.bfloat16()), "float32"), (dict(z=x[:2]), "shape"),
                          (dict(keep=torch.ones(16, dtype=torch.uint8, device="cuda")), "keep"), (dict(keep=x), "keep"), (dict(pre=(ones[:8], None)), "pre gamma"),
                          (dict(pre=(None, ones)), "gamma"), (dict(post=(ones, ones.half())), "post beta"), (dict(pre=(ones, None), res_scale=ones.half()), "float16"),
                          (dict(norm="batch"), "norm"), (dict(eps=-1.0), "eps"), (dict(eps=math.nan), "eps"), (dict(u=x.cpu()), "GPU"), (dict(res_scale=ones.double()), "float32")):
        with pytest.raises((ValueError, RuntimeError), match=match):
            ops.gated_residual_norm(x, **kwargs)
    with pytest.raises(ValueError, match="8192"):
        ops.gated_residual_norm(torch.zeros(2, 8193, device="cuda"))
    with pytest.raises(ValueError, match="8192"):
        ops.gated_residual_norm(torch.zeros(2, 0, device="cuda"))
    with pytest.raises(RuntimeError, match="float32"):
        ops.gated_residual_norm(x.double())


# ------------------------------------------------------------------------------------------------ gradient clipping
def _gradients(g, sizes, types):
    return [(0.1 * _randn(g, *(s if isinstance(s, tuple) else (s,)))).to(types[i % len(types)]) for i, s in enumerate(sizes)]


CLIP = [([1], [F32]), ([7], [BF16]), ([0, 3, 0, 8193, 0], [F32]), ([(64, 5), 5, (128, 64), 128, 1], [F32, BF16, F16]), ([8192, 8191, 16385, 100003], [F16]),
        ([3] * 500, [F32]), ([(i * 37) % 300 for i in range(481)], [F32, F16, BF16]), ([3_000_001, 17, 2_500_000], [F32]), ([9_000_003], [BF16]),
        ([160 * 8192 + 5] + [1] * 320, [F32])]


@pytest.mark.parametrize("p", [1.0, 2.0, math.inf])
@pytest.mark.parametrize("case", range(len(CLIP)))
def test_clip_grad_norm(ops, case, p):
    sizes, types = CLIP[case]
    g = _gen(case)
    grads = _gradients(g, sizes, types)
    norm, bound, _, _ = clip_reference(grads, 1.0, p)
    for factor in (0.3, 5.0):
        max_norm = factor * float(norm)
        _, _, want, bounds = clip_reference(grads, max_norm, p)
        dev = [t.cuda() for t in grads]
        got = ops.global_grad_norm(dev, p)
        assert got.shape == () and got.dtype == F32
        check(got, norm, bound, "norm alone")
        out = [torch.full_like(t, 7.0) for t in dev]
        got = ops.clip_grad_norm_(dev, max_norm, p, out=out)
        check(got, norm, bound, "norm")
        for i, (o, t, d) in enumerate(zip(out, grads, dev)):
            check(o, want[i], bounds[i], f"output {i}")
            assert torch.equal(d.cpu(), t), "an input was written"
            assert factor < 1 or torch.equal(o, d), "within max_norm the values stay"
        again = ops.clip_grad_norm_(dev, max_norm, p)
        assert torch.equal(again, got)
        for d, o in zip(dev, out):
            assert torch.equal(d, o), "in place and into an output differ"


def test_clip_grad_norm_layouts_and_lists(ops):
    """Gradients as slices of one buffer at any address, transposed ones, generators, None entries, an empty list, a zero limit."""
    g = _gen(20)
    flat = _randn(g, 5000).cuda()
    sizes = [1, 2, 3, 5, 1000, 1, 777, 64, 3]
    views, at = [], 1
    for s in sizes:
        views.append(flat[at:at + s])
        at += s
    host = [v.cpu().clone() for v in views]
    norm, bound, want, bounds = clip_reference(host, 2.0, 2.0)
    before = flat.clone()
    versions = [v._version for v in views]
    got = ops.clip_grad_norm_((v for v in views), 2.0)
    check(got, norm, bound, "norm")
    for i, v in enumerate(views):
        check(v, want[i], bounds[i], f"slice {i}")
        assert v._version > versions[i], "a write that autograd cannot see"
    assert torch.equal(flat[:1], before[:1]) and torch.equal(flat[at:], before[at:]), "values next to the slices were written"
    turned = _randn(g, 40, 30).cuda().t()
    turned4 = _randn(g, 2, 3, 4, 5).cuda().permute(2, 0, 3, 1)
    norm, bound, want, bounds = clip_reference([turned, turned4], 1.0, 2.0)
    got = ops.clip_grad_norm_([None, turned, None, turned4], 1.0)
    check(got, norm, bound, "norm")
    check(turned, want[0], bounds[0], "transposed")
    check(turned4, want[1], bounds[1], "permuted")
    assert float(ops.clip_grad_norm_([], 1.0)) == 0 and float(ops.global_grad_norm([None])) == 0
    assert float(ops.clip_grad_norm_([torch.zeros(0, device="cuda")], 1.0)) == 0
    zero = torch.zeros(100, device="cuda")
    assert float(ops.clip_grad_norm_([zero], 1.0)) == 0 and not bool(zero.any())
    kept = turned4.clone()
    with torch.inference_mode():
        frozen = torch.ones(5, device="cuda")
    with pytest.raises(RuntimeError, match="nference"):
        ops.clip_grad_norm_([turned4, frozen], 1e-3)
    assert torch.equal(turned4, kept)
    kept[0, 0, 0, 0] = math.inf
    before = kept.clone()
    assert float(ops.clip_grad_norm_([kept], math.inf)) == math.inf and torch.equal(kept, before)
    ops.clip_grad_norm_([turned], 0.0)
    assert not bool(turned.any())


@pytest.mark.parametrize("p", [1.0, 2.0, math.inf])
def test_clip_grad_norm_non_finite_and_extreme_values(ops, p):
    big = torch.full((1000,), 1e30).cuda()
    norm, bound, want, bounds = clip_reference([big], 1.0, p)
    check(ops.global_grad_norm([big], p), norm, bound, "squares beyond fp32")
    ops.clip_grad_norm_([big], 1.0, p)
    check(big, want[0], bounds[0], "clipped")
    a, b = torch.ones(5000).cuda(), torch.ones(9).cuda()
    a[4999] = -math.inf
    assert float(ops.clip_grad_norm_([a, b], 1.0, p)) == math.inf
    assert not bool(b.any()) and not bool(a[:4999].any()) and bool(torch.isnan(a[4999]))
    a, b = torch.ones(5000, dtype=BF16).cuda(), torch.ones(9).cuda()
    a[17], a[18] = math.nan, math.inf
    assert math.isnan(float(ops.clip_grad_norm_([a, b], 1.0, p)))
    assert bool(torch.isnan(a).all()) and bool(torch.isnan(b).all())
    small = torch.full((300,), 1e-42).cuda()                     # below the smallest normal number
    norm, bound, _, _ = clip_reference([small], 1.0, p)
    check(ops.global_grad_norm([small], p), norm, bound + tiny(F32), "subnormal")


def test_clip_grad_norm_refusals(ops):
    a = torch.ones(100, device="cuda")
    for grads, kwargs, match in (([a, a], {}, "invalid"), ([a[:60], a[50:]], {}, "invalid"), ([a.expand(3, 100)], {}, "densely"), ([a[::2]], {}, "densely"),
                                 ([a.double()], {}, "float32"), ([a, a.cpu()], {}, "one GPU"), ([a.clone().requires_grad_(True)], {}, "requires"),
                                 ([a], dict(out=[a[:50]]), "output"), ([a], dict(out=[a.half()]), "output"), ([a[:50]], dict(out=[a[1:51]]), "invalid"),
                                 ([a.view(10, 10)], dict(out=[torch.ones(10, 10, device="cuda").t()]), "output")):
        with pytest.raises((ValueError, RuntimeError), match=match):
            ops.clip_grad_norm_(grads, 1.0, **kwargs)
    assert torch.equal(a, torch.ones_like(a))
    check(ops.global_grad_norm([a, a]), torch.tensor(200.0, dtype=torch.float64).sqrt(), 20 * U, "reading the same tensor twice is fine")


# ------------------------------------------------------------------------------------------------ streams, graphs, neighbours
def _training_pass(ops, ids, table, block, grads_out, max_norm):
    """Class ids -> table rows -> gated block -> gradients -> clipped: the operators in the order of a training step."""
    x = ops.embedding(ids, table, 2.0)
    y, n = ops.gated_residual_norm(x, None, block["z"], post=block["post"], res_scale=block["scale"], pre=block["pre"])
    leaves = [table, block["z"], block["scale"], *block["post"], *block["pre"]]
    grads = torch.autograd.grad([y, n], leaves, [block["dy"], block["dn"]])
    norm = ops.clip_grad_norm_(grads, max_norm, out=grads_out)
    return [y.detach(), n.detach(), norm, *grads_out]


def _training_state(seed, rows=9000, V=300, D=72):
    g = _gen(seed)
    ids = _ids(g, rows, V, "hot", torch.int32).cuda()
    table = _randn(g, V, D).cuda().requires_grad_(True)
    block = {k: _device(v) for k, v in _block(g, (rows, D), F32, F32, False, True, False, True, True, True, "layer").items() if k in ("z", "post", "scale", "pre")}
    block["dy"], block["dn"] = _randn(g, rows, D).cuda(), _randn(g, rows, D).cuda()
    leaves = [table, block["z"], block["scale"], *block["post"], *block["pre"]]
    return ids, table, block, [torch.empty_like(t) for t in leaves]


def test_training_pass_of_the_three_operators(ops):
    """The chain against 64 bits: autograd through the formulas.  Relative error in the 2-norm: four fp32 norms and a few hundred rows a
    sum, each a few u times its condition (below 100 for these rows): 1e-5 leaves a factor of ten."""
    ids, table, block, outs = _training_state(30)
    got = _training_pass(ops, ids, table, block, outs, 1.0)
    t64 = table.detach().double().cpu().requires_grad_(True)
    leaf = {k: block[k].detach().double().cpu().requires_grad_(True) for k in ("z", "scale")}
    post, pre = ([v.detach().double().cpu().requires_grad_(True) for v in block[k]] for k in ("post", "pre"))
    pad = torch.cat((t64, torch.zeros(1, 72, dtype=torch.float64)))
    i = ids.cpu().long()
    x = 2.0 * pad[torch.where(i < 0, 300, i)]
    ln = torch.nn.functional.layer_norm
    y = x + leaf["scale"] * torch.sigmoid(leaf["z"]) * ln(x, (72,), post[0], post[1], 1e-5)
    n = ln(y, (72,), pre[0], pre[1], 1e-5)
    grads = torch.autograd.grad([y, n], [t64, leaf["z"], leaf["scale"], *post, *pre], [block["dy"].double().cpu(), block["dn"].double().cpu()])
    norm = torch.cat([v.reshape(-1) for v in grads]).norm()
    want = [y.detach(), n.detach(), norm, *(v / (norm + 1e-6) for v in grads)]
    for k, (a, b) in enumerate(zip(got, want)):
        a = a.double().cpu()
        assert float((a - b).norm()) <= 1e-5 * float(b.norm()), f"output {k}: {float((a - b).norm() / b.norm()):.2e}"


def test_captured_and_replayed(ops):
    """Two graphs of the training pass, captured one after the other and replayed in turn with eager work between: every replay equals the
    eager result on the inputs that are in place then."""
    states = [_training_state(40 + k, rows=r, V=v, D=d) for k, (r, v, d) in enumerate(((3000, 40, 64), (9000, 700, 33)))]
    eager = [[t.clone() for t in _training_pass(ops, *s, 1.0)] for s in states]
    graphs, outputs = [], []
    for s in states:
        ids, table, block, outs = s
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            _training_pass(ops, *s, 1.0)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            captured = _training_pass(ops, *s, 1.0)
        graphs.append(graph)
        outputs.append(captured)
    for turn in range(3):
        for k in (0, 1):
            if turn == 2:                                     # new inputs in the captured places
                with torch.no_grad():
                    states[k][2]["dy"].mul_(-0.5)
                    states[k][0].copy_(states[k][0].flip(0))
                eager[k] = [t.clone() for t in _training_pass(ops, *states[k], 1.0)]
            for t in outputs[k]:
                t.zero_()
            torch.cuda.synchronize()
            graphs[k].replay()
            ops.global_grad_norm([states[1 - k][2]["dy"]])
            torch.cuda.synchronize()
            for i, (a, b) in enumerate(zip(outputs[k], eager[k])):
                assert torch.equal(a, b), f"graph {k}, turn {turn}, output {i}"


def test_two_streams_at_once(ops):
    """The same calls on two streams that run next to each other give what they give alone."""
    states = [_training_state(50 + k) for k in range(2)]
    alone = [[t.clone() for t in _training_pass(ops, *s, 1.0)] for s in states]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in states]
    for turn in range(4):
        got = []
        for st in streams:
            st.wait_stream(torch.cuda.current_stream())
        for s, st in zip(states, streams):
            with torch.cuda.stream(st):
                got.append(_training_pass(ops, *s, 1.0))
        torch.cuda.synchronize()
        for k in range(2):
            for a, b in zip(got[k], alone[k]):
                assert torch.equal(a, b), f"stream {k}, turn {turn}"


def test_outputs_end_where_they_end(ops):
    """Nothing is written behind a tensor's last value: outputs through the C entries into the middle of a larger buffer."""
    from mbvae_amd import _lib
    g = _gen(60)
    st = torch.cuda.current_stream().cuda_stream
    for dtype, code in ((F32, 0), (BF16, 1), (F16, 2)):
        for rows, D in ((1, 1), (3, 77), (5, 130), (2, 1037), (33, 9)):
            guard, size = 64, rows * D
            buf = torch.full((size + 2 * guard,), 3.0, dtype=dtype, device="cuda")
            mid = buf[guard:guard + size]
            x = _randn(g, rows, D, dtype=dtype).cuda()
            ids = torch.randint(0, rows, (rows,), generator=g).cuda()
            _lib.call("mbvae_embedding_fwd", ids.data_ptr(), 8, x.data_ptr(), mid.data_ptr(), rows, rows, D, 1.0, code, st)
            assert torch.equal(mid.view(rows, D), x[ids]) and bool((buf[:guard] == 3).all()) and bool((buf[guard + size:] == 3).all())
            ws = torch.empty(_lib.query("mbvae_embedding_bwd_workspace", rows, rows, D, code), dtype=torch.uint8, device="cuda")
            _lib.call("mbvae_embedding_bwd", ids.data_ptr(), 8, x.data_ptr(), D, mid.data_ptr(), rows, rows, D, 1.0, code, ws.data_ptr(), ws.numel(), st)
            check(mid.view(rows, D), *embedding_gradient(ids, x, rows, 1.0), "dweight")
            assert bool((buf[:guard] == 3).all()) and bool((buf[guard + size:] == 3).all())
            ones = torch.ones(D, device="cuda")
            nbuf = buf.clone()
            _lib.call("mbvae_gated_norm_fwd", x.data_ptr(), D, 0, 0, 0, 0, 0, 1.0, 0, 0, 0, ones.data_ptr(), 0, mid.data_ptr(), nbuf[guard:].data_ptr(), 0, rows, D,
                      0, 1e-5, code, 0, st)
            for b in (buf, nbuf):
                assert bool((b[:guard] == 3).all()) and bool((b[guard + size:] == 3).all())
            assert half_step(dtype) > 0


# ------------------------------------------------------------------------------------------------ where the framework uses them
def _close(a, b, rel, what):
    """Relative error in the 2-norm."""
    a, b = a.detach().double().cpu(), b.detach().double().cpu()
    assert a.shape == b.shape and bool(torch.isfinite(a).all()), what
    assert float((a - b).norm()) <= rel * float(b.norm()), f"{what}: {float((a - b).norm() / b.norm()):.2e}"


@pytest.mark.parametrize("which", ["residual", "transformer", "fusion"])
@pytest.mark.parametrize("bias,dropout", [(True, 0.0), (True, 0.1), (False, 0.1)])
def test_fused_blocks_of_the_encoders(ops, which, bias, dropout):
    """Encoders and fusion with the fused updates against the separate kernels: the same dropout masks from the same generator, outputs and
    all gradients to fp32 rounding.  The chain is 3 layers of norms, products of up to 256 terms and gates; a rounding of 2^-24 a step grows by
    the layers' condition, a few hundred steps of it stay below 1e-5 - but for ReLU gates that flip, none of which these inputs have
    within rounding (checked by the bound itself)."""
    from mbvae_amd import blocks
    torch.manual_seed(5)
    if which == "fusion":
        net = blocks.CrossAttentionFusion(64, 32, 3, factor=4, dropout=dropout, bias=bias).cuda().train()
        inputs = [torch.randn(40, 64).cuda().requires_grad_(True) for _ in range(2)]
    else:
        cls = blocks.ResidualEncoder if which == "residual" else blocks.TransformerEncoder
        net = cls(100, 64, 48, 3, factor=4, dropout=dropout, bias=bias).cuda().train()
        inputs = [torch.randn(40, 100).cuda().requires_grad_(True)]
    leaves = inputs + list(net.parameters())

    def run(fused):
        ops.set_fused_blocks(fused)
        try:
            torch.manual_seed(6)
            out = net(*inputs)
            out = out if torch.is_tensor(out) else out[0]
            state = torch.cuda.get_rng_state()
            return out, torch.autograd.grad(out.square().sum(), leaves, allow_unused=True), state
        finally:
            ops.set_fused_blocks(False)

    want, wg, ws = run(False)
    got, gg, gs = run(True)
    assert torch.equal(ws, gs), "the generator has advanced differently"
    _close(got, want, 1e-5, "output")
    names = [f"input {i}" for i in range(len(inputs))] + [k for k, _ in net.named_parameters()]
    for k, a, b in zip(names, gg, wg):
        assert (a is None) == (b is None), k
        if a is not None:
            _close(a, b, 1e-5, k)
    net.eval()
    with torch.no_grad():
        ops.set_fused_blocks(True)
        got = net(*inputs)
        ops.set_fused_blocks(False)
        want = net(*inputs)
    for a, b in zip(got if isinstance(got, tuple) else [got], want if isinstance(want, tuple) else [want]):
        _close(a, b, 1e-5, "evaluation")


def _small_denoiser():
    from mbvae_amd.graph_transformer import GraphTransformer
    torch.manual_seed(7)
    return GraphTransformer(n_layers=2, input_dims={"X": 13, "E": 5, "y": 77}, hidden_mlp_dims={"X": 32, "E": 16, "y": 64},
                            hidden_dims={"dx": 64, "de": 16, "dy": 64, "n_head": 4, "dim_ffX": 32, "dim_ffE": 16, "dim_ffy": 64},
                            output_dims={"X": 5, "E": 5, "y": 64}).cuda()


@pytest.mark.parametrize("id_dtype", [torch.int8, torch.int64])
def test_denoiser_from_edge_classes(ops, id_dtype):
    """GraphTransformer.forward with the pairs' classes against the one-hot rows alone: outputs and all gradients to fp32 rounding (the edge
    input MLP sees the same rows; only the order in which its gradients are summed differs)."""
    from mbvae_amd.trainstep import synthetic_graphs
    net = _small_denoiser()
    g = _gen(8)
    bs, n = 5, 12
    X0, E0, mask = synthetic_graphs(bs, n, "cuda", g, sizes=torch.tensor([12, 9, 1, 12, 3]))
    E0 = E0 * (mask.unsqueeze(1) & mask.unsqueeze(2)).unsqueeze(-1)
    ids = torch.where(E0.sum(-1) > 0, E0.argmax(-1), -1).to(id_dtype)
    X, y = torch.cat((X0, torch.randn(bs, n, 8, generator=g).cuda()), 2), torch.randn(bs, 77, generator=g).cuda()
    w = [torch.randn(*s, generator=g).cuda() for s in ((bs, n, 5), (bs, n, n, 5))]

    def run(**kw):
        out = net(X, E0, y, mask, **kw)
        params = [p for k, p in net.named_parameters() if "mlp_out_y" not in k]
        return out, torch.autograd.grad((out.X * w[0]).sum() + (out.E * w[1]).sum(), params, allow_unused=True)

    for train in (False, True):
        net.train(train)
        for layer in net.tf_layers:
            layer.dropout_p = 0.0                       # (dropout draws from the seeds' order, which is the same; off for the comparison)
        want, wg = run()
        got, gg = run(edge_ids=ids)
        _close(got.X, want.X, 1e-5, "X")
        _close(got.E, want.E, 1e-5, "E")
        for (k, _), a, b in zip([(k, p) for k, p in net.named_parameters() if "mlp_out_y" not in k], gg, wg):
            if b is not None and float(b.norm()) > 1e-4:
                _close(a, b, 2e-5, k)
    net.eval()
    with torch.no_grad():
        for _ in range(2):                              # (the second call takes the packed path where the widths allow it)
            want, got = net(X, E0, y, mask), net(X, E0, y, mask, edge_ids=ids)
            _close(got.E, want.E, 1e-5, "E without gradients")
    for bad in (ids[..., :-1], ids.float(), ids > 0):
        with pytest.raises(ValueError, match="edge_ids"):
            net(X, E0, y, mask, edge_ids=bad)


def test_train_step_with_classes_and_clipping(ops):
    """DenoiserTrainStep with edge_classes and max_grad_norm: the same loss as without, the gradients' norm as torch computes it, and the
    update of clipped gradients."""
    from mbvae_amd.trainstep import CFG3, DenoiserTrainStep, synthetic_graphs
    cfg = {**CFG3, "n_layers": 1, "hidden_mlp_dims": {"X": 32, "E": 16, "y": 64}, "input_dims": {"X": 13, "E": 5, "y": 77}, "output_dims": {"X": 5, "E": 5, "y": 64},
           "hidden_dims": {"dx": 64, "de": 16, "dy": 64, "n_head": 4, "dim_ffX": 32, "dim_ffE": 16, "dim_ffy": 64}}
    g = _gen(9)
    X0, E0, mask = synthetic_graphs(8, 16, "cuda", g, sizes=torch.randint(2, 17, (8,), generator=g))
    cond = torch.randn(8, 64, generator=g).cuda()

    def run(**kw):
        step = DenoiserTrainStep(cfg=cfg, side_stream=False, **kw)
        for layer in step.model.tf_layers:
            layer.dropout_p = 0.0
        taken = []
        update = step.opt.step

        def spy(*a, **k):
            taken.append([p.grad.clone() for p in step.model.parameters() if p.grad is not None])
            return update(*a, **k)

        step.opt.step = spy
        torch.manual_seed(10)
        loss = step.step(X0, E0, mask, cond)
        return loss, taken[0], step.last

    loss, grads, last = run()
    assert "grad_norm" not in last
    total = torch.linalg.vector_norm(torch.cat([t.double().reshape(-1) for t in grads]))
    for kw in (dict(max_grad_norm=0.1 * float(total)), dict(edge_classes=True, max_grad_norm=0.1 * float(total))):
        l2, g2, last = run(**kw)
        _close(l2, loss, 1e-6, "loss")
        _close(last["grad_norm"], total, 2e-5, "norm")
        _close(torch.linalg.vector_norm(torch.cat([t.double().reshape(-1) for t in g2])), 0.1 * total, 2e-5, "clipped norm")


def test_lightning_gradient_clipping_hook(ops):
    from mbvae_amd.abstract import AbstractDTIModel
    model = AbstractDTIModel()
    model.lin = torch.nn.Linear(8, 4).cuda()
    model.unused = torch.nn.Parameter(torch.zeros(3).cuda())
    opt = torch.optim.SGD(model.parameters(), lr=0.1)

    def grads():
        opt.zero_grad()
        (model.lin(torch.ones(5, 8, device="cuda")).sum() * 3).backward()
        return [p.grad for p in model.lin.parameters()]

    before = [t.clone() for t in grads()]
    norm = torch.cat([t.reshape(-1) for t in before]).double().norm()
    model.configure_gradient_clipping(opt, None)
    model.configure_gradient_clipping(opt, 0.0, "norm")
    assert all(torch.equal(a, p.grad) for a, p in zip(before, model.lin.parameters())) and "train/grad_norm" not in model.logged
    model.configure_gradient_clipping(opt, 0.5)
    for a, p in zip(before, model.lin.parameters()):
        check(p.grad, a.double() * (0.5 / (norm + 1e-6)), (a.double() * 0.5 / norm).abs() * 4 * U, "clipped by norm")
    check(model.logged["train/grad_norm"], norm, float(norm) * 2 * U, "logged norm")
    grads()
    model.configure_gradient_clipping(opt, 2.0, "value")
    assert all(float(p.grad.abs().max()) <= 2.0 for p in model.lin.parameters())
    with pytest.raises(ValueError, match="gradient_clip_algorithm"):
        model.configure_gradient_clipping(opt, 1.0, "other")


# ------------------------------------------------------------------------------------------------ past 32 bits
FAR = (1 << 22) + 3                  # rows of 1024 values: the last ones lie behind 2^32 values and 2^33 bytes


def _far_rows(seed):
    """[FAR, 1024] bf16, every row its own: a row of noise scaled by a value that differs from its neighbours'."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    row = torch.randn(1024, generator=g, device="cuda").bfloat16()
    factor = (torch.rand(FAR, 1, generator=g, device="cuda") + 0.5).bfloat16()
    return row * factor


LOOK = [0, 1, FAR // 2, (1 << 21) - 1, 1 << 21, (1 << 22) - 1, 1 << 22, FAR - 2, FAR - 1]


def test_embedding_past_32_bits(ops):
    table = _far_rows(1)
    ids = torch.tensor([0, FAR - 1, 1 << 22, FAR - 1, 7, (1 << 21) + 5, FAR, -1], device="cuda")
    got = ops.embedding(ids, table, 2.0)
    want, bound = embedding_reference(torch.arange(6), torch.stack([table[i] for i in ids[:6].tolist()]), 2.0)
    check(got[:6], want, bound, "far rows of the table")
    assert not bool(got[6:].any())
    weight = table.requires_grad_(True)
    dy = torch.randn(8, 1024, device="cuda").bfloat16()
    dw, = torch.autograd.grad(ops.embedding(ids, weight), weight, dy)
    want, bound = embedding_gradient(torch.tensor([0, 1, 2, 1, 3, 4]), dy[:6], 5, 1.0)
    check(dw[torch.tensor([0, FAR - 1, 1 << 22, 7, (1 << 21) + 5], device="cuda")], want, bound, "far rows of its gradient")
    assert int(dw.any(1).sum()) == 5
    del table, weight, dw
    # as many tokens: few classes, then enough of them for the sort
    dy = _far_rows(2)
    for classes in (3, 40):
        ids = (torch.arange(FAR, device="cuda") % (classes + 1)).to(torch.int8)          # (one id in classes + 1 is outside the table)
        w = torch.randn(classes, 1024, device="cuda").bfloat16().requires_grad_(True)
        y = ops.embedding(ids, w)
        for r in LOOK:
            k = r % (classes + 1)
            assert torch.equal(y[r], w.detach()[k] if k < classes else torch.zeros_like(y[r]))
        dw, = torch.autograd.grad(y, w, dy)
        for k in (0, classes - 1):
            mine = dy[k::classes + 1]
            total = sum(mine[i:i + (1 << 18)].double().sum(0) for i in range(0, mine.shape[0], 1 << 18))
            size = sum(mine[i:i + (1 << 18)].double().abs().sum(0) for i in range(0, mine.shape[0], 1 << 18))
            check(dw[k], total, total.abs() * half_step(BF16) + size * U * 4096, "a class's gradient")      # (sums of at most 1024 by 4096 terms)
        del y, dw


def test_gated_residual_norm_past_32_bits(ops):
    x, z = _far_rows(3), _far_rows(4)
    gamma, beta = torch.ones(1024, device="cuda"), torch.zeros(1024, device="cuda")
    dy = _far_rows(5)
    leaves = [x.requires_grad_(True), z.requires_grad_(True)]
    y, n = ops.gated_residual_norm(x, None, z, pre=(gamma, beta))
    dx, dz = torch.autograd.grad([y, n], leaves, [dy, dy])
    pick = torch.tensor(LOOK, device="cuda")
    few = dict(x=x.detach()[pick], u=None, z=z.detach()[pick], keep=None, keep_scale=1.0, post=None, scale=None, pre=(gamma, beta), norm="layer")
    want = gated_reference(**few, eps=1e-5, dy=dy[pick], dn=dy[pick])
    for k, t in (("y", y), ("n", n), ("dx", dx), ("dz", dz)):
        check(t[pick], *want[k], k)


def test_clip_grad_norm_past_32_bits(ops):
    big = _far_rows(6)
    small = torch.ones(3, device="cuda")
    norm = ops.global_grad_norm([small, big])
    total = sum(big[i:i + (1 << 18)].double().square().sum() for i in range(0, FAR, 1 << 18)) + 3
    check(norm, total.sqrt(), float(total.sqrt()) * 2 * U, "norm")
    pick = torch.tensor(LOOK, device="cuda")
    before = big[pick].double()
    ops.clip_grad_norm_([small, big], 0.25 * float(norm))
    check(big[pick], before * 0.25, before.abs() * (half_step(BF16) + 8 * U), "clipped")


@pytest.mark.parametrize("V,D", [((1 << 21) + 3, 1024), ((1 << 22) + 3, 1024), ((1 << 20) + 1, 3 * 1024 + 5), (131075, 16385)])
@pytest.mark.parametrize("rows", [0, 7])
def test_embedding_gradient_clears_tables_past_32_bits(ops, rows, V, D):
    """Every row of the table's gradient that no token has is written, whatever lay in its place: tables just past 2^31 and 2^32 values and between
    them, through the C entry into memory full of NaN, by the radix sort, by one ordering launch (the last table) and without any token."""
    from mbvae_amd import _lib
    ids = torch.tensor([0, V - 1, 1 << 16, V - 1, 5, V, -1], device="cuda")[:rows]
    dy = torch.randn(rows, D, generator=_gen(D)).bfloat16().cuda()
    dw = torch.full((V, D), math.nan, dtype=BF16, device="cuda")
    ws = torch.empty(max(16, _lib.query("mbvae_embedding_bwd_workspace", rows, V, D, 1)), dtype=torch.uint8, device="cuda")
    _lib.call("mbvae_embedding_bwd", ids.data_ptr(), 8, dy.data_ptr(), D, dw.data_ptr(), rows, V, D, 1.0, 1, ws.data_ptr(), ws.numel(),
              torch.cuda.current_stream().cuda_stream)
    if rows:
        want, bound = embedding_gradient(torch.tensor([0, 1, 2, 1, 3]), dy[:5], 4, 1.0)
        taken = torch.tensor([0, V - 1, 1 << 16, 5], device="cuda")
        check(dw[taken], want, bound, "rows with tokens")
        dw[taken] = 0
    for r in range(0, V, 1 << 18):
        assert not bool(dw[r:r + (1 << 18)].any()), f"rows {r} to {r + (1 << 18)} hold values that nobody has written"


@pytest.mark.parametrize("D,dtype", [(5, F32), (64, F32), (300, BF16), (512, F32), (520, BF16), (1037, F32), (4100, F32)])
def test_gated_residual_norm_rows_whose_squares_leave_fp32(ops, D, dtype):
    """A row of finite values whose mean square is beyond fp32 normalises to 0, as in the separate LayerNorm kernel (n is beta exactly, the
    norm passes no gradient on); one infinity in a row takes only itself with it under the root mean square.  Other rows do not notice."""
    g = _gen(D)
    x, u = _randn(g, 9, D), _randn(g, 9, D)
    x[3], x[7], u[4] = x[3] * 1e25, -3e24, u[4] * 1e25
    x, u = x.to(dtype), u.to(dtype)
    gamma, beta, dy, dn = 1 + 0.2 * _randn(g, D), _randn(g, D), _randn(g, 9, D, dtype=dtype), _randn(g, 9, D, dtype=dtype)
    gamma, beta = gamma.cuda(), beta.cuda()
    for norm in ("layer", "rms"):
        leaves = [t.cuda().requires_grad_(True) for t in (x, u)]
        y, n = ops.gated_residual_norm(*leaves, post=(gamma, beta), pre=(gamma, beta), norm=norm)
        dx, du = torch.autograd.grad([y, n], leaves, [dy.cuda(), dn.cuda()])
        assert bool(torch.isfinite(y).all()) and bool(torch.isfinite(n).all()) and bool(torch.isfinite(dx).all()) and bool(torch.isfinite(du).all())
        assert not bool(du[4].any()) and torch.equal(dx[3].cpu(), dy[3]), "a norm without scale passes no gradient on"
        want = beta.to(dtype)
        assert torch.equal(n[3], want) and torch.equal(y[4], (x[4].cuda().float() + beta).to(dtype))
        if norm == "rms":                                  # (a row of equal values has no spread: LayerNorm sees a mean square within range)
            assert torch.equal(n[7], want)
        for i in (0, 1, 2, 5, 6, 8):
            few = dict(x=x[i:i + 1], u=u[i:i + 1], z=None, keep=None, keep_scale=1.0, post=(gamma, beta), scale=None, pre=(gamma, beta), norm=norm)
            ref = gated_reference(**few, eps=1e-5, dy=dy[i:i + 1], dn=dn[i:i + 1])
            for k, t in (("y", y), ("n", n), ("dx", dx), ("du", du)):
                check(t[i:i + 1], *ref[k], f"{k}, row {i}")
    if dtype == F32:
        plain = ops.ln_residual(x.cuda(), None, gamma, beta)
        _, n = ops.gated_residual_norm(x.cuda(), torch.zeros_like(x).cuda(), pre=(gamma, beta))
        assert torch.equal(torch.isnan(n), torch.isnan(plain)) and torch.equal(n[3], plain[3])
    row = _randn(g, 2, D, dtype=dtype)
    row[0, D // 2] = math.inf
    _, n = ops.gated_residual_norm(row.cuda(), torch.zeros_like(row).cuda(), pre=(gamma, None), norm="rms")
    rest = torch.arange(D, device="cuda") != D // 2
    assert bool(torch.isnan(n[0, D // 2])) and not bool(n[0, rest].any()) and bool(torch.isfinite(n[1]).all())


def test_forward_mode_is_refused(ops):
    """An operand with a tangent: an error, not a result whose tangent is gone - whether or not anything also asks for a reverse pass."""
    import torch.autograd.forward_ad as forward_ad
    g = _gen(70)
    ids = torch.tensor([0, 2, 1], device="cuda")
    host = _block(g, (3, 8), F32, F32, True, True, False, True, True, True, "layer")
    dev = {k: _device(v, False) if k not in ("keep_scale", "norm") else v for k, v in host.items()}
    plain = torch.ones(3, 8, device="cuda")
    with forward_ad.dual_level():
        def dual(t):
            return forward_ad.make_dual(t.detach(), torch.ones_like(t))

        for leaf in (False, True):
            with pytest.raises(RuntimeError, match="forward-mode"):
                ops.embedding(ids, dual(plain.clone().requires_grad_(leaf)))
            for k, b in ([(k, {**dev, k: dual(dev[k])}) for k in ("x", "u", "z", "scale")]
                         + [(k, {**dev, k: pair}) for k in ("post", "pre") for pair in ((dual(dev[k][0]), dev[k][1]), (dev[k][0], dual(dev[k][1])))]):
                b["z"] = b["z"].requires_grad_(leaf) if k != "z" else b["z"]
                with pytest.raises(RuntimeError, match="forward-mode"):
                    _call(ops, b, 1e-5)
                b["z"].requires_grad_(False)
        with pytest.raises(RuntimeError, match="forward-mode"):
            ops.global_grad_norm([plain, dual(plain)])
        with pytest.raises(RuntimeError, match="forward-mode"):
            ops.clip_grad_norm_([dual(plain.clone())], 1.0)
        with pytest.raises(RuntimeError, match="forward-mode"):
            ops.clip_grad_norm_([plain], 1.0, out=[dual(plain.clone())])
        assert ops.embedding(ids, plain).shape == (3, 8) and bool((plain == 1).all())
    y, n = _call(ops, dev, 1e-5)
    assert bool(torch.isfinite(n).all())


@pytest.mark.parametrize("p", [1.0, 2.0, math.inf])
@pytest.mark.parametrize("dtype,value,max_norm", [(F32, 3e38, 1e-3), (F32, -3e38, 1e-12), (BF16, 2e38, 1e-2), (F32, 3e38, 1.0), (F32, 1e-3, 1e-38), (F16, 6e4, 1e-35)])
def test_clip_grad_norm_by_a_factor_below_fp32(ops, dtype, value, max_norm, p):
    """A factor max_norm / norm below the smallest normal fp32 number keeps its bits: outputs to the same bound as any other."""
    grads = [torch.full((1000,), value, dtype=dtype), torch.linspace(-1, 1, 777).to(dtype) * value, torch.zeros(5, dtype=dtype)]
    _, _, want, bounds = clip_reference(grads, max_norm, p)
    dev = [t.cuda() for t in grads]
    out = [torch.full_like(t, 7.0) for t in dev]
    ops.clip_grad_norm_(dev, max_norm, p, out=out)
    ops.clip_grad_norm_(dev, max_norm, p)
    for i, (o, d) in enumerate(zip(out, dev)):
        check(o, want[i], bounds[i], f"output {i}")
        assert torch.equal(o, d), "in place and into an output differ"


@pytest.mark.parametrize("V,dtype", [(16, F32), (16, BF16), (40, F16)])
def test_embedding_of_the_widest_rows(ops, V, dtype):
    """Rows of 2^23 values: few classes and many."""
    D = 1 << 23
    dy = torch.randn(3, D, device="cuda").to(dtype)
    ids = torch.tensor([0, V - 1, V - 1], device="cuda")
    weight = torch.randn(V, D, device="cuda").to(dtype).requires_grad_(True)
    y = ops.embedding(ids, weight)
    assert torch.equal(y, weight.detach()[ids])
    dw, = torch.autograd.grad(y, weight, dy)
    assert torch.equal(dw[0], dy[0]) and torch.equal(dw[V - 1], (dy[1].float() + dy[2].float()).to(dtype)) and not bool(dw[1:V - 1].any())


def test_embedding_forward_past_one_side_of_a_grid(ops):
    """2^26 rows of 516 values take 2^24 blocks of 256 threads: more than one side of a grid holds."""
    rows, D = 1 << 26, 516
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < rows * D * 4 + (8 << 30):
        pytest.skip("138 GB of output do not fit")
    ids = (torch.arange(rows, device="cuda") % 7 - 1).to(torch.int8)
    table = torch.randn(5, D, device="cuda")
    padded = torch.cat((torch.zeros(1, D, device="cuda"), table, torch.zeros(1, D, device="cuda")))
    y = ops.embedding(ids, table)
    for r in range(0, rows, 1 << 20):
        assert torch.equal(y[r:r + (1 << 20)], padded[ids[r:r + (1 << 20)].long() + 1]), f"rows from {r}"
    del y
    torch.cuda.empty_cache()


@pytest.mark.parametrize("kind", ["kernels", "strided", "float64", "two places", "history"])
def test_lightning_hook_by_kernels_and_by_torch(ops, kind):
    """On the GPU the hook takes the kernels where they take the gradients and torch where they do not; the result is the same function."""
    from mbvae_amd.abstract import AbstractDTIModel
    g = _gen(80)
    grads = [_randn(g, 40, 6).cuda(), _randn(g, 9).cuda(), _randn(g, 3, 4)[:, ::2].cuda()]
    if kind == "strided":
        grads.append(_randn(g, 50, 8).cuda()[:, ::2])
    elif kind == "float64":
        grads[1] = grads[1].double()
    elif kind == "two places":
        grads[0] = grads[0].cpu()
    elif kind == "history":
        grads[0] = grads[0].requires_grad_(True) * 1.0
    model = AbstractDTIModel()
    for i, t in enumerate(grads):
        p = torch.nn.Parameter(torch.zeros(t.shape, dtype=t.dtype, device=t.device))
        p.grad = t
        model.register_parameter(f"p{i}", p)
    model.register_parameter("unused", torch.nn.Parameter(torch.zeros(2, device="cuda")))
    assert ops.clip_grad_norm_takes([p.grad for p in model.parameters()]) == (kind == "kernels")
    want = [t.detach().double().cpu().clone() for t in grads]
    norm = math.sqrt(sum(float(t.square().sum()) for t in want))
    model.configure_gradient_clipping(torch.optim.SGD(model.parameters(), lr=0.1), 0.25 * norm)
    for p, t in zip(model.parameters(), want):
        check(p.grad, 0.25 * t, 0.25 * t.abs() * 16 * U, "clipped")        # (torch: an fp32 norm of a few hundred squares, a quotient, a product)
    assert abs(float(model.logged["train/grad_norm"]) - norm) <= 16 * U * norm


def test_kernel_calls_are_noted_while_profiling(ops):
    """_lib.PROFILE sees the calls of these operators as it sees all others, the backward's (issued from autograd's thread) among them, and
    from the moment it is set on."""
    from mbvae_amd import _lib
    state = _training_state(90, rows=500)
    plain = [t.clone() for t in _training_pass(ops, *state, 1.0)]
    y = ops.embedding(state[0], state[1])
    noted = {}
    try:
        _lib.PROFILE = noted
        assert _lib.PROFILE is noted
        y.sum().backward()
        assert [k for k, _ in noted] == ["mbvae_embedding_bwd"]
        got = _training_pass(ops, *state, 1.0)
        ops.dense_from_ids(torch.zeros(1, 4, dtype=torch.int8, device="cuda"), torch.zeros(1, 4, 4, dtype=torch.int8, device="cuda"), 5, 5)
        with pytest.raises(RuntimeError, match="invalid"):
            ops.clip_grad_norm_([y.detach(), y.detach()], 1.0)
    finally:
        _lib.PROFILE = None
    _training_pass(ops, *state, 1.0)
    torch.cuda.synchronize()
    assert {k: len(v) for (k, _), v in noted.items()} == {"mbvae_embedding_fwd": 1, "mbvae_embedding_bwd": 2, "mbvae_gated_norm_fwd": 1,
                                                          "mbvae_gated_norm_bwd": 1, "mbvae_grad_clip": 1, "mbvae_dense_from_ids": 1}
    assert all(0 < start.elapsed_time(end) < 1000 for calls in noted.values() for start, end in calls)
    for a, b in zip(got, plain):
        assert torch.equal(a, b)


@pytest.mark.parametrize("D", [1, 7, 64, 1037])
@pytest.mark.parametrize("ptype", [F32, BF16, F16])
def test_gradients_of_a_blocks_vectors_lie_apart_and_aligned(ops, D, ptype):
    """They share one allocation: each begins at 16 bytes, ends where it ends, and writing one leaves the others."""
    host = _block(_gen(D), (6, D), F32, ptype, True, False, False, True, True, True, "layer")
    dev = {k: _device(v) if k not in ("keep_scale", "norm") else v for k, v in host.items()}
    y, n = _call(ops, dev, 1e-5)
    vectors = [dev["scale"], *dev["post"], *dev["pre"]]
    (y.sum() + n.square().sum()).backward()
    grads = [v.grad for v in vectors]
    assert all(t.data_ptr() % 16 == 0 and t.is_contiguous() and t.shape == (D,) for t in grads)
    before = [t.clone() for t in grads]
    for i, t in enumerate(grads):
        t.fill_(float(i))
    assert all(bool((t == i).all()) for i, t in enumerate(grads)) and all(bool(torch.isfinite(t).all()) for t in before)
    ops.clip_grad_norm_(grads, 0.5)                       # (refused if any two of them met)


def test_clip_grad_norm_refused_leaves_no_trace(ops):
    """A refused call has not written, and autograd is not told that it has: what was saved for a backward pass is still good."""
    leaf = torch.ones(100, device="cuda", requires_grad=True)
    a = torch.full((100,), 3.0, device="cuda")
    y = leaf * a
    for grads, kwargs in (([a, a], {}), ([a[:60], a[50:]], {}), ([a, torch.ones(100, device="cuda")], dict(out=[torch.ones(100, device="cuda"), a]))):
        versions = a._version
        with pytest.raises(RuntimeError, match="invalid"):
            ops.clip_grad_norm_(grads, 1.0, **kwargs)
        assert a._version == versions
    y.sum().backward()
    assert torch.equal(leaf.grad, a)
    y = leaf * a
    ops.clip_grad_norm_([a], 1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.sum().backward()
    with torch.inference_mode():
        frozen = torch.full((100,), 3.0, device="cuda")
        ops.clip_grad_norm_([frozen], 1.0)
    assert float(frozen[0]) < 1
    with pytest.raises(RuntimeError, match="nference"):
        ops.clip_grad_norm_([torch.ones(100, device="cuda")], 1e-3, out=[frozen])


@pytest.mark.parametrize("size", [1e-9, 1e-7, 1e-3, 0.5, 3.0, 1e4])
def test_clip_grad_norm_at_its_limit(ops, size):
    """Limits on both sides of the norm: values stay bit for bit exactly where norm + 1e-6 <= max_norm, but for a factor that rounds to 1, and
    follow the formula where the 1e-6 is all that there is (a norm of 1e-9 and a limit of 1e-7: a tenth)."""
    g = _gen(95)
    t = _randn(g, 5000)
    t = t * (size / float(t.double().norm()))
    norm = float(t.double().norm())
    for max_norm in (norm, norm * (1 - 1e-3), norm * (1 + 1e-3), norm + 1e-6, math.nextafter(norm + 1e-6, math.inf), norm + 2e-6, 0.5 * norm, 1e-7, 1e-6):
        _, _, want, bounds = clip_reference([t], max_norm, 2.0)
        dev = t.cuda()
        ops.clip_grad_norm_([dev], max_norm)
        check(dev, want[0], bounds[0], f"limit {max_norm}")
        factor = max_norm / (norm + 1e-6)
        if factor >= 1 + 1e-12:                                        # (the norm's own last bits decide at 1)
            assert torch.equal(dev.cpu(), t), f"limit {max_norm}: within the limit the values stay"
        elif factor < 1 - 2 * U:
            assert not torch.equal(dev.cpu(), t), f"limit {max_norm}: above the limit the values are scaled"


def test_fused_blocks_wider_than_the_kernel(ops):
    """Hidden widths above 8192 run with the fused updates switched on as well: by the separate kernels, bit for bit."""
    from mbvae_amd import blocks
    torch.manual_seed(5)
    for cls in (blocks.TransformerEncoder, blocks.ResidualEncoder):
        net = cls(12, ops.GATED_NORM_MAX_WIDTH + 8, 4, 1, factor=1, dropout=0.1).cuda().train()
        x = torch.randn(3, 12, device="cuda")
        got = []
        for fused in (False, True):
            ops.set_fused_blocks(fused)
            try:
                torch.manual_seed(6)
                got.append(net(x))
            finally:
                ops.set_fused_blocks(False)
        assert torch.equal(got[0], got[1])


def test_operands_that_are_marked_as_negated(ops):
    """The imaginary part of a conjugate is a view of values with the other sign: every operand in turn against its materialised twin."""
    g = _gen(100)

    def marked(*shape):
        t = torch.view_as_complex(_randn(g, *shape, 2).cuda()).conj().imag
        assert t.is_neg()
        return t

    for D in (1, 6):
        host = _block(g, (5, D), F32, F32, True, True, False, True, True, True, "layer")
        plain = {k: _device(v, False) if k not in ("keep_scale", "norm") else v for k, v in host.items()}
        for k in ("x", "u", "z", "scale", "post", "pre"):
            shape = (5, D) if k in ("x", "u", "z") else (D,)
            t = marked(*shape)
            twin = t.clone().resolve_neg()
            if k in ("post", "pre"):
                pairs = [((t, plain[k][1]), (twin, plain[k][1])), ((plain[k][0], t), (plain[k][0], twin))]
            else:
                pairs = [(t, twin)]
            for a, b in pairs:
                for got, want in zip(_call(ops, {**plain, k: a}, 1e-5), _call(ops, {**plain, k: b}, 1e-5)):
                    assert torch.equal(got, want), (k, D)
        x = plain["x"].clone().requires_grad_(True)
        y, n = _call(ops, {**plain, "x": x}, 1e-5)
        dy = marked(5, D)
        a, = torch.autograd.grad(y, x, dy, retain_graph=True)
        b, = torch.autograd.grad(y, x, dy.clone().resolve_neg())
        assert torch.equal(a, b)
        ids, table = torch.tensor([0, 3, 3], device="cuda"), marked(4, D)
        assert torch.equal(ops.embedding(ids, table), table.clone().resolve_neg()[ids])
        w = plain["x"][:4].clone().requires_grad_(True)
        y, dy = ops.embedding(ids, w), marked(3, D)
        assert torch.equal(torch.autograd.grad(y, w, dy, retain_graph=True)[0], torch.autograd.grad(y, w, dy.clone().resolve_neg())[0])
    t = torch._neg_view(torch.arange(1.0, 9.0, device="cuda"))
    norm = ops.global_grad_norm([t])
    check(norm, torch.tensor(204.0, dtype=torch.float64).sqrt(), 30 * U, "norm")
    with pytest.raises(ValueError, match="sign"):
        ops.clip_grad_norm_([t], 1.0, out=[torch.zeros(8, device="cuda")])
    before = t.clone().resolve_neg()
    ops.clip_grad_norm_([t], 0.5 * float(norm))
    check(t, before.double() * 0.5, before.abs() * 8 * U, "clipped in place")


@pytest.mark.parametrize("rows,V,D,dtype", [(16384, 5, 1024, F32), (16384, 5, 1025, F32), (16353, 5, 1025, F32), (40000, 5, 1024, BF16), (40000, 5, 1028, BF16),
                                            (32768, 32, 160, F32), (32768, 32, 161, F32), (33000, 16, 512, BF16), (4096, 32, 640, F32), (4096, 32, 641, F32),
                                            (100, 32, 20000, F32), (8, 1, 1 << 20, F16), (3, 2, (1 << 21) - 1, F32), (16384, 2, 4096, BF16),
                                            (16384, 3, 4096, BF16)])
def test_embedding_gradient_where_the_routes_meet(ops, rows, V, D, dtype):
    """Few classes on both sides of the table size from which they are ordered.  A workspace is never as large as dy but for the smallest."""
    from mbvae_amd import _lib
    g = _gen(rows + D)
    ids, dy = _ids(g, rows, V, "hot", torch.int8), _randn(g, rows, D, dtype=dtype)
    weight = torch.zeros(V, D, dtype=dtype, device="cuda", requires_grad=True)
    y = ops.embedding(ids.cuda(), weight, 0.5)
    dw, = torch.autograd.grad(y, weight, dy.cuda(), retain_graph=True)
    check(dw, *embedding_gradient(ids, dy, V, 0.5), "dweight")
    assert torch.equal(torch.autograd.grad(y, weight, dy.cuda())[0], dw)
    size = rows * D * dy.element_size()
    code = {F32: 0, BF16: 1, F16: 2}[dtype]
    assert _lib.query("mbvae_embedding_bwd_workspace", rows, V, D, code) <= max(22 << 20, size // 2)


def test_embedding_gradient_workspace_stays_small(ops):
    """Many rows of few, wide classes: the blocks' tables are bounded, whatever the rows."""
    from mbvae_amd import _lib
    for code, most in ((0, 32), (1, 16), (2, 16)):
        for rows in (1000, 32768, 1 << 20, (1 << 31) - 1):
            for V in (1, 5, most):
                for D in (64, 512, 5120, 65536, 1 << 23):
                    dy = rows * D * (4 if code == 0 else 2)
                    assert _lib.query("mbvae_embedding_bwd_workspace", rows, V, D, code) <= max(22 << 20, dy // 3 + 20 * rows), (code, rows, V, D)


def test_clip_grad_norm_leaves_tensor_subclasses_to_torch(ops):
    """Gradients that only look like tensors in memory (a distributed tensor is one) are not the kernels' to take."""
    class Wrapped(torch.Tensor):
        @staticmethod
        def __new__(cls, inner):
            return torch.Tensor._make_wrapper_subclass(cls, inner.shape, dtype=inner.dtype, device=inner.device, strides=inner.stride())

        @classmethod
        def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
            raise NotImplementedError(str(func))

    plain = torch.ones(8, device="cuda")
    assert ops.clip_grad_norm_takes([plain]) and not ops.clip_grad_norm_takes([plain, Wrapped(plain)])
