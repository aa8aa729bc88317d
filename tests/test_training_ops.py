"""The training-side operators (geodiffuser_amd.ops / .training: token embedding, block norms, gradient clipping) against plain
implementations in 64 bits, at the sizes, layouts and values where they can go wrong, and their refusals.

Tolerances, derived before any run.  Storage of type T rounds a result r by at most u |r| with u = finfo(T).eps / 2, or half its smallest
subnormal (``_close``).  The arithmetic before that rounding is binary32 (2^-24 relative a step); a result that is a sum of terms t_i
built by at most k roundings on any path is then off by at most k 2^-24 sum |t_i|.  Each check states its k and its sum of magnitudes."""
import ctypes
import math

import pytest
import torch

from geodiffuser_amd import GeodiffError

gpu = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.float16, torch.bfloat16, torch.float32]
U32 = 2.0 ** -24


@pytest.fixture(scope="module")
def ops():
    from geodiffuser_amd import _lib, ops as _ops
    _lib.load()
    return _ops


def _gen(seed):
    return torch.Generator(device="cpu").manual_seed(seed)


def _randn(g, *shape, dtype=torch.float32, std=1.0, mean=0.0, dev=DEV):
    return (torch.randn(*shape, generator=g) * std + mean).to(dev).to(dtype)


def _close(got, ref, k, mag, what=""):
    """|got - ref| <= u |ref| + half a subnormal + k 2^-24 mag, NaN and infinities where ref has them."""
    fi = torch.finfo(got.dtype)
    u = 0.0 if got.dtype == torch.float32 else fi.eps / 2
    got, ref = got.double(), ref.double()
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    fine = ref.isfinite()
    assert torch.equal(got.isnan(), ref.isnan()) and torch.equal(got[~fine & ~ref.isnan()], ref[~fine & ~ref.isnan()]), what
    err = (got - ref).abs()
    tol = (u * (1 + u) + U32) * ref.abs() + fi.smallest_normal * fi.eps / 2 + k * U32 * mag.double()
    bad = (err > tol) & fine
    if bool(bad.any()):
        i = int((err - tol).masked_fill(~bad, -1).argmax())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off, worst at {i}: {float(got.flatten()[i])} for {float(ref.flatten()[i])}, "
                             f"tolerance {float(tol.expand_as(err).flatten()[i])}")


def _misaligned(t):
    """The same values at an address that is a multiple of the element only."""
    return torch.cat([t.new_zeros(1), t.flatten()])[1:].view(t.shape)


# ------------------------------------------------------------------------------------------------ token embedding
def _embed_ref(ids, table, pos, scale):
    V = table.shape[0]
    ok = (ids >= 0) & (ids < V)
    y = table.double()[ids.long().clamp(0, V - 1)] * scale
    if pos is not None:
        y = y + pos.double()[:ids.shape[-1]]
    return torch.where(ok[..., None], y, torch.nan)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape,V,C,pos,scale", [
    ((1, 1), 5, 8, True, 1.0), ((1,), 3, 1, False, 2.0), ((2, 77), 49408, 1024, True, 1.0), ((3, 5), 100, 333, True, 333 ** 0.5), ((2, 3, 7), 9, 1280, False, 0.5),
    ((1, 77), 1000, 2056, True, 1.0), ((513, 9), 4000, 40, True, -3.0), ((4, 2), 1, 65, True, 1.0)])
def test_embedding_lookup(ops, dtype, shape, V, C, pos, scale):
    g = _gen(C)
    ids = torch.randint(0, V, shape, generator=g)
    ids.view(-1)[-1] = V - 1
    table, P = _randn(g, V, C, dtype=dtype), _randn(g, shape[-1] + 2, C, dtype=dtype) if pos else None
    ref = _embed_ref(ids.to(DEV), table, P, scale)
    mag = (table.double()[ids.to(DEV)] * scale).abs() + (0 if P is None else P.double()[:shape[-1]].abs())
    for idx in (ids.to(DEV), ids.to(DEV).int()):
        # k = 2: scale itself to 32 bits, the fused multiply-add
        _close(ops.embed_tokens(idx, table, P, scale=scale), ref, 2, mag)
    _close(ops.embed_tokens(ids.to(DEV), _misaligned(table), P, scale=scale), ref, 2, mag)


@gpu
def test_embedding_lookup_outside_the_table_is_nan(ops):
    table = torch.ones(4, 24, device=DEV)
    ids = torch.tensor([[0, -1, 4, 3, -2 ** 40, 2 ** 40]], device=DEV)
    y = ops.embed_tokens(ids, table, torch.ones(6, 24, device=DEV))
    assert torch.equal(y.isnan().all(-1), torch.tensor([[False, True, True, False, True, True]], device=DEV)) and torch.equal(y[0, 0], torch.full((24,), 2.0, device=DEV))
    assert ops.embed_tokens(ids[:, :0], table).shape == (1, 0, 24)


def _check_embed_bwd(ops, ids, dy, V, scale=1.0, padding_idx=None):
    d = ops.embed_tokens_bwd(ids, dy, V, scale=scale, padding_idx=padding_idx)
    flat, rows = ids.reshape(-1).long(), dy.reshape(-1, dy.shape[-1]).double() * scale
    ok = (flat >= 0) & (flat < V)
    if padding_idx is not None:
        ok &= flat != padding_idx
    ref = torch.zeros(V, dy.shape[-1], dtype=torch.float64, device=DEV).index_add_(0, flat[ok], rows[ok])
    mag = torch.zeros_like(ref).index_add_(0, flat[ok], rows[ok].abs())
    # k: the additions of the longest row and the scaling
    k = int(torch.bincount(flat[ok]).max()) + 2 if bool(ok.any()) else 0
    _close(d, ref, k, mag, f"n={flat.numel()} V={V} C={dy.shape[-1]}")
    assert not bool(d[torch.bincount(flat[ok], minlength=V) == 0].any())              # rows of no token: exact zeros
    assert torch.equal(d, ops.embed_tokens_bwd(ids, dy, V, scale=scale, padding_idx=padding_idx))      # and the same bits again


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,V,C,kind", [
    (0, 7, 16, "any"), (1, 1, 1, "any"), (1, 50, 9, "any"), (5, 33, 64, "same"), (77, 1000, 768, "prompt"), (255, 17, 24, "any"), (256, 300, 512, "any"),
    (257, 300, 520, "distinct"), (308, 49408, 1024, "prompt"), (1000, 40, 333, "any"), (1500, 2000, 1280, "distinct"), (3000, 5, 128, "any"),
    (4096, 100, 40, "same"), (4097, 49408, 96, "prompt"), (20011, 1003, 136, "prompt"), (20000, 3, 64, "any"), (9999, 70000, 72, "distinct"), (70001, 500, 33, "any")])
def test_embedding_gradient(ops, dtype, n, V, C, kind):
    g = _gen(n + C)
    if kind == "same":
        ids = torch.full((n,), V // 2)
    elif kind == "distinct":
        ids = torch.randperm(max(n, V), generator=g)[:n] % V
    elif kind == "prompt":
        ids = (V * torch.rand(n, generator=g) ** 5).long()
        ids[torch.rand(n, generator=g) < 0.6] = 0
    else:
        ids = torch.randint(0, V, (n,), generator=g)
    dy = _randn(g, n, C, dtype=dtype)
    _check_embed_bwd(ops, ids.to(DEV), dy, V)
    _check_embed_bwd(ops, ids.to(DEV).int(), _misaligned(dy) if n else dy, V, scale=0.125)


@gpu
@pytest.mark.parametrize("n", [1030, 9000, 70000, 140000, 300000])
@pytest.mark.parametrize("seed", range(4))
def test_embedding_gradient_of_every_run_length(ops, n, seed):
    """Tokens that occur just as often as fills, ends at, goes one over a tile of 8 .. 64 sorted entries, two tiles, many."""
    g = _gen(seed)
    lengths = [1, 2, 7, 8, 9, 15, 16, 17, 24, 31, 32, 33, 48, 63, 64, 65, 127, 128, 129, 192, 193, 257, 1025, 5000]
    counts = []
    while sum(counts) < n:
        counts.append(lengths[int(torch.randint(0, len(lengths) if seed else 12, (1,), generator=g))])
    counts[-1] -= sum(counts) - n
    ids = torch.repeat_interleave(torch.arange(len(counts)) * 2, torch.tensor(counts))[torch.randperm(n, generator=g)].to(DEV)
    _check_embed_bwd(ops, ids, _randn(g, n, 24), 2 * len(counts))
    _check_embed_bwd(ops, ids, _randn(g, n, 9, dtype=torch.bfloat16), 2 * len(counts), padding_idx=2 * len(counts) - 2)


@gpu
@pytest.mark.parametrize("n,V", [(900, 1 << 21), (2000, (1 << 20) + 7), (2000, (1 << 20) - 1), (4097, 255), (4096, 256), (5000, 65535), (5000, 65536), (30000, 3000001), (3000, (1 << 24) + 3)])
def test_embedding_gradient_of_large_vocabularies(ops, n, V):
    """Tokens of one to four bytes: as many passes of the sort, and the one-launch sort's limit on either side."""
    g = _gen(n)
    ids = torch.randint(0, V, (n,), generator=g)
    ids[::3] = V - 1
    ids[1::7] = ids[0]
    _check_embed_bwd(ops, ids.to(DEV), _randn(g, n, 8), V)
    _check_embed_bwd(ops, ids.to(DEV), _randn(g, n, 3, dtype=torch.float16), V, padding_idx=V - 1)


@gpu
@pytest.mark.parametrize("n", [6, 300, 9000])
def test_embedding_gradient_skips_padding_and_foreign_ids(ops, n):
    g = _gen(n)
    ids = torch.randint(-2, 8, (3, n // 3), generator=g).to(DEV)                      # -2, -1, 6, 7 lie outside a table of 6 rows
    dy = _randn(g, *ids.shape, 40)
    for pad in (None, 0, 5):
        _check_embed_bwd(ops, ids, dy, 6, padding_idx=pad)
    ids[ids == 3] = 2 ** 40                                                            # beyond 32 bits
    _check_embed_bwd(ops, ids, dy, 6)
    _check_embed_bwd(ops, torch.full_like(ids, -1), dy, 6)                             # nothing inside: all zeros


@gpu
def test_embedding_gradient_keeps_nan_and_inf_in_their_rows(ops):
    for n in (40, 8000):
        ids = (torch.arange(n) % 8).to(DEV)
        dy = torch.ones(n, 16, device=DEV)
        dy[1, 2], dy[2, 3] = math.nan, math.inf
        d = ops.embed_tokens_bwd(ids, dy, 9)
        want = torch.full((9, 16), n / 8, device=DEV)
        want[8] = 0
        want[1, 2], want[2, 3] = math.nan, math.inf
        assert torch.equal(d.nan_to_num(nan=-1, posinf=-2), want.nan_to_num(nan=-1, posinf=-2))


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lead,L,P,C", [((1,), 1, 1, 8), ((4,), 77, 77, 1024), ((2, 3), 5, 9, 33), ((0,), 3, 4, 16), ((1000,), 7, 77, 40), ((3001,), 2, 3, 520)])
def test_position_gradient(ops, dtype, lead, L, P, C):
    dy = _randn(_gen(L), *lead, L, C, dtype=dtype)
    d = ops.embed_positions_bwd(dy, P)
    rows = dy.double().reshape(-1, L, C)
    pad = torch.zeros(P - L, C, dtype=torch.float64, device=DEV)
    _close(d, torch.cat([rows.sum(0), pad]), rows.shape[0], torch.cat([rows.abs().sum(0), pad]))        # k: one addition a sequence
    assert not bool(d[L:].any()) and torch.equal(d, ops.embed_positions_bwd(dy, P))
    if dy.numel():
        assert rel_same(ops.embed_positions_bwd(_misaligned(dy), P), d, rows.shape[0], rows.abs().sum(0).max())


def rel_same(a, b, k, mag):
    """Two results of the same sums in possibly different orders."""
    u = 0.0 if a.dtype == torch.float32 else torch.finfo(a.dtype).eps
    return bool(((a.double() - b.double()).abs() <= u * b.double().abs() + 2 * k * U32 * mag + torch.finfo(a.dtype).smallest_normal).all())


@gpu
def test_embedding_offsets_beyond_32_bits(ops):
    """A table and a gradient of more than 2^31 elements: the rows behind that border are the ones asked for."""
    V, C = (1 << 21) + 5, 1024
    table = torch.zeros(V, C, dtype=torch.bfloat16, device=DEV)
    table[-1], table[-3] = 3.0, 5.0
    ids = torch.tensor([[V - 1, V - 3, 0]], device=DEV)
    assert ops.embed_tokens(ids, table)[0, :, 7].tolist() == [3.0, 5.0, 0.0]
    d = ops.embed_tokens_bwd(ids, torch.ones(1, 3, C, dtype=torch.bfloat16, device=DEV), V)
    assert d[[V - 1, V - 3, 0, V - 2], C - 1].tolist() == [1.0, 1.0, 1.0, 0.0] and float(d.sum(dtype=torch.float32)) == 3.0 * C
    del d
    ids = torch.zeros(V, dtype=torch.int32, device=DEV)                               # the same buffer as the gradient of as many positions
    ids[-1], ids[-3] = 2, 1
    d = ops.embed_tokens_bwd(ids, table, 4)
    assert d[:, 5].tolist() == [0.0, 5.0, 3.0, 0.0]
    assert ops.embed_positions_bwd(table.view(1, V, C), V)[-1, 0].item() == 3.0


def test_embedding_refusals():
    from geodiffuser_amd import ops
    t, ids = torch.zeros(4, 8), torch.zeros(2, 3, dtype=torch.long)
    for call in (lambda: ops.embed_tokens(ids, t), lambda: ops.embed_tokens_bwd(ids, torch.zeros(2, 3, 8), 4), lambda: ops.embed_positions_bwd(torch.zeros(2, 3, 8), 3)):
        with pytest.raises(GeodiffError, match="GPU tensor"):
            call()


@gpu
def test_embedding_refusals_on_the_device(ops):
    t, ids, dy = torch.zeros(4, 8, device=DEV), torch.zeros(2, 3, dtype=torch.long, device=DEV), torch.zeros(2, 3, 8, device=DEV)
    bad = [lambda: ops.embed_tokens(ids.cpu(), t), lambda: ops.embed_tokens(ids.float(), t), lambda: ops.embed_tokens(ids.short(), t), lambda: ops.embed_tokens(ids, t.double()),
           lambda: ops.embed_tokens(ids, t.t()), lambda: ops.embed_tokens(ids.t(), t), lambda: ops.embed_tokens(ids, t, t[:2]), lambda: ops.embed_tokens(ids, t, t.half()),
           lambda: ops.embed_tokens(ids, t, torch.zeros(4, 9, device=DEV)), lambda: ops.embed_tokens(ids, t, t.cpu()), lambda: ops.embed_tokens(ids[0, 0], t),
           lambda: ops.embed_tokens_bwd(ids, dy[:1], 4), lambda: ops.embed_tokens_bwd(ids, dy, 4, padding_idx=4), lambda: ops.embed_tokens_bwd(ids, dy, 4, padding_idx=-1),
           lambda: ops.embed_tokens_bwd(ids, dy.double(), 4), lambda: ops.embed_positions_bwd(dy, 2), lambda: ops.embed_tokens(ids, torch.zeros(0, 8, device=DEV))]
    for i, call in enumerate(bad):
        with pytest.raises(GeodiffError):
            call()
            pytest.fail(str(i))


# ------------------------------------------------------------------------------------------------ block norms
EPS = 1e-5


def _norm64(v, kind, gamma, beta, eps):
    """-> (output, xh, r, magnitudes of what a value of xh is made of)."""
    mean = v.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(v[..., :1])
    r = ((v - mean).pow(2).mean(-1, keepdim=True) + eps).rsqrt()
    xh = (v - mean) * r
    y = xh if gamma is None else xh * gamma
    return (y if beta is None else y + beta), xh, r


def _block_ref(x, res, pre, post, gate, res_scale, gy=None, gs=None):
    """Values and magnitudes (sums of the absolute values of all terms) of the forward and of the gradients, in 64 bits."""
    d = lambda t: None if t is None else t.double()
    X, R, G = d(x), d(res), d(gate)
    if G is not None and G.dim() == 2 and x.dim() > 2:
        G = G.view(G.shape[0], *([1] * (x.dim() - 2)), G.shape[1])
    one = lambda t, like: torch.ones_like(like) if t is None else d(t).expand_as(like)
    v, m = {}, {}
    if post is not None:
        h, xh, xr = _norm64(X, post.kind, d(post.gamma), d(post.beta), post.eps)
        # an error of the mean or the values reaches xh as (|v| + mean |v|) r, one of r as |xh|
        mxh = (X.abs() + X.abs().mean(-1, keepdim=True)) * xr + xh.abs()
        mh = mxh * one(post.gamma, X).abs() + (0 if post.beta is None else d(post.beta).abs())
    else:
        h, mh = X, X.abs()
    s = h if G is None else G * h
    ms = mh if G is None else G.abs() * mh
    if R is not None:
        s, ms = s + res_scale * R, ms + abs(res_scale) * R.abs()
    v["s"], m["s"] = s, ms
    if pre is not None:
        y, sh, sr = _norm64(s, pre.kind, d(pre.gamma), d(pre.beta), pre.eps)
        # the sum's own error (its magnitude) enters the mean and the deviation too
        msh = (ms + ms.mean(-1, keepdim=True)) * sr + sh.abs() * (1 + (ms * sh.abs()).mean(-1, keepdim=True) * sr)
        v["y"], m["y"] = y, msh * one(pre.gamma, X).abs() + (0 if pre.beta is None else d(pre.beta).abs())
    if gy is None and gs is None:
        return v, m
    lead = tuple(range(x.dim() - 1))
    over = lambda t, dims: t.sum(dims) if dims else t                # (torch sums over everything for no dimensions)
    ds, mds = torch.zeros_like(s), torch.zeros_like(s)
    if gy is not None:
        g = d(gy) * one(pre.gamma, X)
        gm = g.mean(-1, keepdim=True) if pre.kind == "layer" else 0.0
        ds = sr * (g - gm - sh * (g * sh).mean(-1, keepdim=True))
        ga = g.abs()
        mds = sr * (ga + ga.mean(-1, keepdim=True) + msh * (ga * sh.abs()).mean(-1, keepdim=True) + sh.abs() * (ga * msh).mean(-1, keepdim=True))
        mds = mds + ds.abs() * (1 + (ms * sh.abs()).mean(-1, keepdim=True) * sr)
        v["dpre_gamma"], m["dpre_gamma"] = over(d(gy) * sh, lead), over(d(gy).abs() * msh, lead)
        v["dpre_beta"], m["dpre_beta"] = over(d(gy), lead), over(d(gy).abs(), lead)
    if gs is not None:
        ds, mds = ds + d(gs), mds + d(gs).abs()
    v["dres"], m["dres"] = res_scale * ds, abs(res_scale) * mds
    dh, mdh = ds, mds
    if G is not None:
        dims = lead if gate.dim() == 1 else tuple(range(1, x.dim() - 1))
        v["dgate"], m["dgate"] = over(ds * h, dims), over(mds * h.abs() + ds.abs() * mh, dims)
        dh, mdh = G * ds, G.abs() * mds
    if post is not None:
        v["dpost_gamma"], m["dpost_gamma"] = over(dh * xh, lead), over(mdh * xh.abs() + dh.abs() * mxh, lead)
        v["dpost_beta"], m["dpost_beta"] = over(dh, lead), over(mdh, lead)
        gam = one(post.gamma, X)
        g, mg = dh * gam, mdh * gam.abs()
        gm = g.mean(-1, keepdim=True) if post.kind == "layer" else 0.0
        dh = xr * (g - gm - xh * (g * xh).mean(-1, keepdim=True))
        mdh = xr * (mg + mg.mean(-1, keepdim=True) + mxh * (g * xh).abs().mean(-1, keepdim=True) + xh.abs() * (mg * xh.abs() + g.abs() * mxh).mean(-1, keepdim=True))
        mdh = mdh + dh.abs() * (1 + (X.abs() * xh.abs()).mean(-1, keepdim=True) * xr)
    v["dx"], m["dx"] = dh, mdh
    return v, m


# roundings on any path of one row's arithmetic: 16 channels a thread, 6 + 16 additions across threads, and fewer than 30 in the formulas
K_ROW = 64


def _check_block(ops, x, res, pre, post, gate, res_scale, gy, gs):
    s, y, stats = ops.block_norm(x, res, pre, post=post, gate=gate, res_scale=res_scale)
    v, m = _block_ref(x, res, pre, post, gate, res_scale, gy, gs)
    _close(s, v["s"], K_ROW, m["s"], "s")
    if pre is None:
        assert y is None
    else:
        _close(y, v["y"], K_ROW, m["y"], "y")
    if gy is None and gs is None:
        return
    d = ops.block_norm_bwd(x, res, gy, gs, stats, pre, post=post, gate=gate, res_scale=res_scale)
    rows = x.numel() // x.shape[-1]
    there = dict(dx=x, dres=res, dgate=gate, dpost_gamma=post and post.gamma, dpost_beta=post and post.beta, dpre_gamma=pre and pre.gamma, dpre_beta=pre and pre.beta)
    for k, t in there.items():
        if t is None:
            assert d[k] is None, k
            continue
        assert d[k].dtype == t.dtype and d[k].shape == t.shape, k
        if gy is None and k.startswith("dpre"):
            assert not bool(d[k].any())
            continue
        # the rows' own arithmetic twice (forward again, backward); sums over rows: one more addition a row at most
        _close(d[k], v[k], 2 * K_ROW + (0 if k in ("dx", "dres") else rows), m[k], k)
    again = ops.block_norm_bwd(x, res, gy, gs, stats, pre, post=post, gate=gate, res_scale=res_scale)
    assert all(t is None or torch.equal(t, again[k]) for k, t in d.items())


def _block_case(ops, shape, dtype, kind, gate, post, res, seed, affine=True, beta=True, strided=False, off=False):
    g = _gen(seed)
    C = shape[-1]
    mis = _misaligned if off else lambda t: t
    norm = lambda kd: ops.Norm(kd, mis(_randn(g, C, dtype=dtype, std=0.2, mean=1.0)) if affine else None,
                               _randn(g, C, dtype=dtype, std=0.2) if affine and beta else None, EPS)
    x = mis(_randn(g, *shape, dtype=dtype, std=0.8, mean=0.3))
    r = _randn(g, *shape, dtype=dtype, std=1.5, mean=-0.2) if res else None
    gt = None
    if gate == "channel":
        gt = _randn(g, C, dtype=dtype, std=0.4, mean=0.7)
    elif gate == "sample":
        gt = _randn(g, shape[0], 3 * C if strided else C, dtype=dtype, std=0.4, mean=0.7)
        gt = gt[:, C:2 * C] if strided else gt
    return x, r, norm(kind), norm("rms" if kind == "layer" and seed % 2 else kind) if post else None, gt, _randn(g, *shape, dtype=dtype), _randn(g, *shape, dtype=dtype, std=0.6)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind,gate,post,res,scale", [
    ("layer", None, False, True, 1.0), ("rms", "sample", True, True, 0.5), ("layer", "channel", True, True, 1.0), ("rms", None, True, False, 1.0),
    ("layer", "sample", False, False, 1.0), ("rms", "channel", False, True, -2.0), ("layer", None, False, False, 1.0)])
@pytest.mark.parametrize("shape", [(1, 1, 8), (1, 77, 1024), (3, 5, 333), (2, 130, 320), (5, 1, 513), (2, 37, 2048)])
def test_block_norm(ops, dtype, kind, gate, post, res, scale, shape):
    x, r, pre, po, gt, gy, gs = _block_case(ops, shape, dtype, kind, gate, post, res, sum(shape))
    _check_block(ops, x, r, pre, po, gt, scale, gy, gs)


@gpu
@pytest.mark.parametrize("C", [1, 2, 7, 64, 65, 512, 520, 1000, 1024, 1025, 1032, 1500, 2056, 4096, 4097, 4104, 8192, 8200, 16383, 16384])
def test_block_norm_widths(ops, C):
    for dtype in (torch.float32, torch.bfloat16):
        x, r, pre, po, gt, gy, gs = _block_case(ops, (2, 6, C), dtype, "layer", "sample", True, True, C)
        _check_block(ops, x, r, pre, po, gt, 1.0, gy, gs)


@gpu
@pytest.mark.parametrize("shape", [(1, 1, 40), (40,), (3, 40), (1, 3, 40), (2, 2, 40), (2, 1023, 40), (700, 3, 40), (2, 3, 4, 5, 40), (1, 5000, 40), (300, 7, 24)])
def test_block_norm_row_counts_and_gate_rows(ops, shape):
    """Rows of one gate that end inside, at and across a workgroup's rows; a 2-d gate beside 2-d activations is a gate for each row."""
    for gate in ("channel", "sample") if len(shape) > 1 else ("channel",):
        x, r, pre, po, gt, gy, gs = _block_case(ops, shape, torch.float32, "rms", gate, True, True, 3)
        _check_block(ops, x, r, pre, po, gt, 1.0, gy, gs)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_block_norm_layouts_and_missing_parts(ops, dtype):
    for C in (96, 333):
        x, r, pre, po, gt, gy, gs = _block_case(ops, (3, 9, C), dtype, "layer", "sample", True, True, 8, strided=True)
        assert not gt.is_contiguous()
        _check_block(ops, x, r, pre, po, gt, 0.7, gy, gs)
        x, r, pre, po, gt, gy, gs = _block_case(ops, (3, 9, C), dtype, "rms", "channel", True, True, 9, off=True)
        _check_block(ops, x, r, pre, po, gt, 0.7, gy, gs)
        x, r, pre, po, gt, gy, gs = _block_case(ops, (3, 9, C), dtype, "layer", "channel", True, True, 10, affine=False)
        _check_block(ops, x, r, pre, po, gt, 1.0, gy, gs)
        x, r, pre, po, gt, gy, gs = _block_case(ops, (3, 9, C), dtype, "layer", None, True, True, 11, beta=False)
        _check_block(ops, x, r, pre, po, gt, 1.0, gy, None)
        _check_block(ops, x, r, pre, po, gt, 1.0, None, gs)
        _check_block(ops, x, r, None, po, gt, 1.0, None, gs)                         # no norm in front of the next block
        _check_block(ops, x, r, None, None, gt, 1.0, None, gs)


@gpu
@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("C", [40, 1024, 3000])
def test_block_norm_hard_values(ops, kind, C):
    """Equal values in a row (variance 0), a zero row, a large mean, large and tiny magnitudes; a NaN and an infinity stay in their rows."""
    g = _gen(C)
    x = _randn(g, 8, C)
    x[0], x[1] = 3.25, 0.0
    x[2] += 1000.0
    x[3] *= 1e15
    x[4] *= 1e-15
    gy, gs = _randn(g, 8, C), _randn(g, 8, C)
    _check_block(ops, x, None, ops.Norm(kind, _randn(g, C), None, 1e-6), None, None, 1.0, gy, gs)
    x[5, 3], x[6, C - 1] = math.nan, math.inf
    n = ops.Norm(kind, None, None, 1e-6)
    s, y, stats = ops.block_norm(x, torch.zeros_like(x), n)
    assert y[[0, 1, 2, 3, 4, 7]].isfinite().all() and y[5].isnan().all() and y[6, C - 1].isnan()
    d = ops.block_norm_bwd(x, torch.zeros_like(x), gy, gs, stats, n)["dx"]
    assert d[[0, 1, 2, 3, 4, 7]].isfinite().all() and d[5].isnan().all()


@gpu
def test_block_norm_beyond_32_bits(ops):
    """Tensors of more than 2^31 elements: the rows behind that border have the bits that a call on them alone gives."""
    R, C = (1 << 21) + 40, 1024
    x = torch.zeros(R, C, dtype=torch.bfloat16, device=DEV)
    tail = _randn(_gen(1), 50, C, dtype=torch.bfloat16)
    x[-50:] = tail
    n = ops.Norm("layer", _randn(_gen(2), C, dtype=torch.bfloat16), None)
    s, y, st = ops.block_norm(x, x, n)
    s2, y2, st2 = ops.block_norm(tail, tail, n)
    assert torch.equal(s[-50:], s2) and torch.equal(y[-50:], y2) and torch.equal(st[-50:], st2) and not bool(y[:50].any())
    del s, y
    d = ops.block_norm_bwd(x, x, x, None, st, n, need=["dx", "dpre_gamma"])
    d2 = ops.block_norm_bwd(tail, tail, tail, None, st2, n, need=["dx", "dpre_gamma"])
    assert torch.equal(d["dx"][-50:], d2["dx"])
    m = (tail.double().abs() * (y2.double().abs() + 1)).sum(0)
    _close(d["dpre_gamma"], d2["dpre_gamma"].double(), 2 * (2 * K_ROW + 50) + 2 ** 17, m)      # each rounds to bf16 once: 2^17 2^-24 = one step of bf16


@gpu
def test_block_norm_need_and_empty(ops):
    x, r, pre, po, gt, gy, gs = _block_case(ops, (2, 33, 64), torch.float32, "layer", "sample", True, True, 5)
    _, _, stats = ops.block_norm(x, r, pre, po, gt)
    full = ops.block_norm_bwd(x, r, gy, gs, stats, pre, po, gt)
    for need in (["dx"], ["dgate"], ["dpre_beta", "dres"], ["dpost_gamma"], []):
        part = ops.block_norm_bwd(x, r, gy, gs, stats, pre, po, gt, need=need)
        for k, t in part.items():
            assert (t is None) == (k not in need) and (t is None or torch.equal(t, full[k])), (k, need)
    e = x[:, :0]
    s, y, stats = ops.block_norm(e, r[:, :0], pre, po, gt)
    assert s.shape == y.shape == e.shape
    d = ops.block_norm_bwd(e, r[:, :0], e, e, stats, pre, po, gt)
    assert d["dx"].shape == e.shape and not bool(d["dgate"].any()) and not bool(d["dpre_gamma"].any())
    s, y, _ = ops.block_norm(x, None, pre)
    assert s is x


@gpu
def test_block_norm_against_differences(ops):
    """<gradient, direction> of the kernel against central differences, of the 64-bit formula and of the kernel's own forward at the same step."""
    g = _gen(77)
    x, r, pre, po, gt, gy, gs = _block_case(ops, (2, 3, 48), torch.float32, "layer", "sample", True, True, 4)
    leaves = dict(dx=x, dres=r, dgate=gt, dpre_gamma=pre.gamma, dpre_beta=pre.beta, dpost_gamma=po.gamma, dpost_beta=po.beta)
    dirs = {k: _randn(g, *t.shape) for k, t in leaves.items()}

    def loss(h, f64):
        c = lambda k, t: (t.double() + h * dirs[k].double()) if f64 else (t + h * dirs[k])
        n, p = ops.Norm(pre.kind, c("dpre_gamma", pre.gamma), c("dpre_beta", pre.beta), EPS), ops.Norm(po.kind, c("dpost_gamma", po.gamma), c("dpost_beta", po.beta), EPS)
        if f64:
            v, _ = _block_ref(c("dx", x), c("dres", r), n, p, c("dgate", gt), 0.5)
            s, y = v["s"], v["y"]
        else:
            s, y, _ = ops.block_norm(c("dx", x), c("dres", r), n, post=p, gate=c("dgate", gt), res_scale=0.5)
        return float((gs.double() * s.double()).sum() + (gy.double() * y.double()).sum())

    _, _, stats = ops.block_norm(x, r, pre, po, gt, 0.5)
    d = ops.block_norm_bwd(x, r, gy, gs, stats, pre, po, gt, 0.5)
    slope = sum(float((d[k].double() * dirs[k].double()).sum()) for k in leaves)
    v, m = _block_ref(x, r, pre, po, gt, 0.5, gy, gs)
    mag = sum(float((m[k] * dirs[k].double().abs()).sum()) for k in leaves)
    h = 2.0 ** -17                                        # truncation ~ h^2 times third derivatives of order 1e3 (rows of deviation ~ 1): below 1e-7 of mag
    assert abs((loss(h, True) - loss(-h, True)) / (2 * h) - slope) <= (2 * K_ROW + 8) * U32 * mag + 1e-6 * mag
    h = 2.0 ** -5                                         # the kernel against the formula at the same points: the outputs' rounding over 2 h
    _, mf = _block_ref(x, r, pre, po, gt, 0.5)
    noise = float((gs.double().abs() * mf["s"]).sum() + (gy.double().abs() * mf["y"]).sum())
    # (x + h d rounds too, by one step: 2 K_ROW covers it; 4: the magnitudes at the moved points)
    assert abs((loss(h, False) - loss(-h, False)) - (loss(h, True) - loss(-h, True))) <= 2 * 4 * 2 * K_ROW * U32 * noise


def test_norm_and_embedding_refusals_on_the_host():
    """The library's own checks, with addresses that are never followed."""
    from geodiffuser_amd import _lib
    lib = _lib.load()
    A = 1 << 20
    ok = dict(x=A, res=A, gate=0, y=A, s=A, stats=A, rows=8, rows_per_gate=8, gate_ld=64, C=64, pre_kind=1, res_scale=1.0)
    bad = [dict(x=0), dict(rows=0), dict(C=0), dict(C=16385), dict(pre_kind=3), dict(post_kind=-1), dict(gate=A, rows_per_gate=3), dict(gate=A, gate_ld=8), dict(gate=A, rows_per_gate=0),
           dict(s=0, y=0, pre_kind=0), dict(pre_kind=0), dict(y=0), dict(rows=1 << 31), dict(gate=A, rows=1 << 17, rows_per_gate=1)]
    for b in bad:
        assert lib.gd_block_norm(ctypes.byref(_lib.GdBlockNorm(**{**ok, **b})), 2, None) < 0, b
    assert lib.gd_block_norm(ctypes.byref(_lib.GdBlockNorm(**ok)), 3, None) == -1 and lib.gd_block_norm(None, 2, None) == -1

    def bwd(f=None, ws=1 << 24, **k):
        return lib.gd_block_norm_bwd(ctypes.byref(_lib.GdBlockNormBwd(f=_lib.GdBlockNorm(**{**ok, **(f or {})}), **k)), ctypes.c_void_p(A), ws, 2, None)

    for k in (dict(), dict(gy=A, f=dict(stats=0)), dict(gy=A, f=dict(pre_kind=0)), dict(gs=A, dpre_gamma=A), dict(gy=A, dpost_gamma=A), dict(gy=A, dgate=A), dict(gy=A, dres=A, f=dict(res=0)),
              dict(gs=A, f=dict(post_kind=2, stats=0))):
        assert bwd(**k) == -1, k
    assert bwd(gy=A, dpre_gamma=A, ws=8) == -2
    nb = lib.gd_embed_bwd_workspace_bytes(5000, 100, 64)
    assert lib.gd_embed_bwd_workspace_bytes(1024, 100, 64) == 0 and nb > 5000 * 16
    E = lambda n=5000, vocab=100, C=64, ids=A, ws=nb, dt=2: lib.gd_embed_bwd(ctypes.c_void_p(ids), 1, n, ctypes.c_void_p(A), vocab, C, -1, 1.0, ctypes.c_void_p(A), ctypes.c_void_p(A), ws, dt, None)
    assert E(n=-1) == -4 and E(n=1 << 30) == -4 and E(vocab=0) == -4 and E(C=0) == -4 and E(ids=0) == -1 and E(ws=nb - 1) == -2 and E(dt=5) == -1
    assert lib.gd_embed(ctypes.c_void_p(A), 1, 0, ctypes.c_void_p(A), 10, None, 1, 8, 1.0, ctypes.c_void_p(A), 2, None) == -1
    assert lib.gd_embed(ctypes.c_void_p(A), 1, 4, ctypes.c_void_p(A), 10, ctypes.c_void_p(A), 0, 8, 1.0, ctypes.c_void_p(A), 2, None) == -1
    assert lib.gd_embed_pos_bwd(ctypes.c_void_p(A), 4, 8, 8, 7, ctypes.c_void_p(A), None, 0, 2, None) == -1
    assert lib.gd_embed_pos_bwd(ctypes.c_void_p(A), 4096, 8, 8, 8, ctypes.c_void_p(A), None, 0, 2, None) == -2


def test_block_norm_refuses_cpu_tensors():
    from geodiffuser_amd import ops
    with pytest.raises(GeodiffError, match="GPU tensor"):
        ops.block_norm(torch.zeros(2, 8), None, ops.Norm("layer"))


@gpu
def test_block_norm_refusals(ops):
    x, n = torch.zeros(2, 3, 8, device=DEV), ops.Norm("layer")
    c = torch.ones(8, device=DEV)
    st = torch.zeros(6, 4, device=DEV)
    big = torch.zeros(1, 16385, device=DEV)
    bad = [lambda: ops.block_norm(x.double(), None, n), lambda: ops.block_norm(x.transpose(0, 1), None, n), lambda: ops.block_norm(x, x[:1], n), lambda: ops.block_norm(x, x.half(), n),
           lambda: ops.block_norm(x, None, None), lambda: ops.block_norm(x, None, ops.Norm("batch")), lambda: ops.block_norm(x, None, ops.Norm("layer", c[:4])),
           lambda: ops.block_norm(x, None, ops.Norm("layer", c.half())), lambda: ops.block_norm(x, None, n, gate=torch.ones(3, 8, device=DEV)),
           lambda: ops.block_norm(x, None, n, gate=torch.ones(8, 2, device=DEV).t()), lambda: ops.block_norm(x, None, n, gate=c.cpu()), lambda: ops.block_norm(big, None, n),
           lambda: ops.block_norm(x, None, n, gate=torch.ones(1, 1, 8, device=DEV)), lambda: ops.block_norm(x, None, n, gate=c[None].expand(2, 8)),
           lambda: ops.block_norm_bwd(x, None, None, None, st, n), lambda: ops.block_norm_bwd(x, x, x, None, st[:5], n), lambda: ops.block_norm_bwd(x, x, x, None, st, None),
           lambda: ops.block_norm_bwd(x, x, x, None, st, n, need=["dy"]), lambda: ops.block_norm_bwd(x, x, x[:1], None, st, n),
           lambda: ops.block_norm(torch.zeros(70000, 8, device=DEV), None, n, gate=torch.ones(70000, 8, device=DEV)), lambda: ops.block_norm(x[..., :0], None, n)]
    for i, call in enumerate(bad):
        with pytest.raises(GeodiffError):
            call()
            pytest.fail(str(i))


# ------------------------------------------------------------------------------------------------ gradient norm and clipping
def _norm_ref(ts, kind=2.0):
    flat = torch.cat([t.double().flatten() for t in ts])
    if kind == 2.0:
        return flat.square().sum().sqrt()
    return flat.abs().max() if flat.numel() else flat.sum()


def _check_clip(ops, ts, max_norm, kind=2.0):
    keep = [t.clone() for t in ts]
    ref = _norm_ref(ts, kind)
    n = ops.grad_norm(ts, kind)
    assert n.shape == () and n.dtype == torch.float32
    # binary64 inside: the conversion to f32 and nothing else that 2^-24 could see
    _close(n, ref, 1, ref)
    assert all(torch.equal(a, b) for a, b in zip(ts, keep))
    f = min(1.0, max_norm / (float(ref) + 1e-6))
    out = [torch.full_like(t, 7.0) for t in ts]
    assert torch.equal(ops.clip_grad_norm(ts, max_norm, kind, out=out), n) and all(torch.equal(a, b) for a, b in zip(ts, keep))
    for t, o in zip(ts, out):
        _close(o, t.double() * f, 2, (t.double() * f).abs())              # the factor to f32, the product
    assert torch.equal(ops.clip_grad_norm(ts, max_norm, kind), n) and all(torch.equal(a, b) for a, b in zip(ts, out))
    return f


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sizes", [(1,), (0, 3, 0), (78848,), (8191, 8192, 8193, 16384, 5), (7, 8, 9, 64, 1000003), (3,) * 127, (11,) * 128, (5,) * 129, tuple(range(300)), (70001,) * 260])
def test_gradient_norm_and_clipping(ops, dtype, sizes):
    for max_norm in (1e-3, 1e6):
        g = torch.Generator(device=DEV).manual_seed(len(sizes))
        ts = [torch.randn(n, generator=g, device=DEV).to(dtype) for n in sizes]
        f = _check_clip(ops, ts, max_norm)
        assert (f < 1) == (max_norm < 1)


@gpu
def test_clipping_mixed_types_and_layouts(ops):
    """Tensors of all three types packed without gaps in a buffer (starts at any multiple of the element), channels_last and 0-d ones."""
    for k in range(3):
        g = _gen(k)
        ts = []
        for dtype in DTYPES:
            sizes = [int(n) for n in torch.randint(1, 40000, (12,), generator=g)]
            flat = _randn(g, sum(sizes), dtype=dtype)
            ts += list(flat.split(sizes))
        ts += [_randn(g, 8, 6, 3, 3, dtype=torch.bfloat16).to(memory_format=torch.channels_last), _randn(g, 1)[0], _randn(g, 5, 0, 3)]
        for kind in (2.0, math.inf):
            _check_clip(ops, [t.clone() if i > 35 else t for i, t in enumerate(ts)], 0.05, kind)


@gpu
def test_clipping_into_buffers_of_another_alignment(ops):
    g = _gen(5)
    for dtype in DTYPES:
        src = [_randn(g, n, dtype=dtype) for n in (1, 100, 8195, 30000)]
        dst = [_misaligned(torch.zeros_like(t)) for t in src]
        n = ops.clip_grad_norm(src, 0.5, out=dst)
        want = [torch.empty_like(t) for t in src]
        ops.clip_grad_norm(src, 0.5, out=want)
        assert all(torch.equal(a, b) for a, b in zip(dst, want)) and float(n) > 0.5
        flat = torch.full((40,), 9.0, device=DEV, dtype=dtype)                    # nothing outside a destination is written
        ops.clip_grad_norm([src[1][:10]], 1e9, out=[flat[15:25]])
        assert torch.equal(flat[15:25], src[1][:10]) and bool((flat[:15] == 9).all()) and bool((flat[25:] == 9).all())


@gpu
def test_gradient_norm_of_extreme_values(ops):
    one = lambda v, dt=torch.float32: torch.full((300,), v, device=DEV, dtype=dt)
    for v in (1e30, 1e-30, 1e-42):                                                # squares beyond the range of f32 on either side
        _close(ops.grad_norm([one(v)]), torch.tensor(float(one(v)[0]) * 300 ** 0.5, dtype=torch.float64, device=DEV), 1, torch.tensor(v, device=DEV))
    _close(ops.grad_norm([one(3e38, torch.bfloat16)]), torch.tensor(math.inf, device=DEV), 0, torch.zeros((), device=DEV))
    t = [one(3e38)]                                                               # a norm above f32's range still clips to max_norm
    assert float(ops.clip_grad_norm(t, 1.0)) == math.inf
    assert abs(float(_norm_ref(t)) - 1.0) < 1e-5
    z = [torch.zeros(10, device=DEV)]
    assert float(ops.clip_grad_norm(z, 1.0)) == 0.0 and not bool(z[0].any())
    assert float(ops.clip_grad_norm([one(2.0)], 0.0)) > 0


@gpu
@pytest.mark.parametrize("kind", [2.0, math.inf])
@pytest.mark.parametrize("where", [0, 8191, 19999])
def test_gradient_norm_of_nan_and_inf(ops, kind, where):
    for count in (1, 200):
        ts = [torch.ones(20000, device=DEV) for _ in range(count)]
        ts[-1][where] = -math.inf
        assert float(ops.grad_norm(ts, kind)) == math.inf
        c = [t.clone() for t in ts]
        assert float(ops.clip_grad_norm(c, 1.0, kind)) == math.inf                 # factor 0, as max / inf is
        assert bool(c[-1][where].isnan()) and float(c[-1].nan_to_num().abs().sum()) == 0
        ts[-1][where] = math.nan
        assert math.isnan(float(ops.grad_norm(ts, kind)))
        ops.clip_grad_norm(ts, 1.0, kind)
        assert all(bool(t.isnan().all()) for t in ts)


@gpu
def test_clipping_beyond_32_bits(ops):
    t = torch.zeros((1 << 31) + 4097, dtype=torch.bfloat16, device=DEV)
    t[-1], t[1 << 31], t[0] = 3.0, 4.0, 12.0
    assert float(ops.clip_grad_norm([t, t.new_full((5,), 0.0)], 6.5)) == 13.0
    assert [float(t[i]) for i in (-1, 1 << 31, 0, 1)] == [1.5, 2.0, 6.0, 0.0]


def test_gradient_norm_refusals_on_the_host():
    """The library's own checks, with addresses that are never followed."""
    from geodiffuser_amd import _lib, ops
    lib = _lib.load()
    with pytest.raises(GeodiffError, match="GPU tensors"):
        ops.grad_norm([torch.zeros(4)])
    with pytest.raises(GeodiffError, match="no tensors"):
        ops.clip_grad_norm([], 1.0)
    with pytest.raises(GeodiffError, match="norm_type"):
        ops.grad_norm([torch.zeros(4)], 1.0)

    def call(src, dst, n, dt, max_norm=1.0, nbytes=1 << 20):
        k = len(src)
        arr = lambda t, v: (t * k)(*v)
        return lib.gd_grad_norm(arr(ctypes.c_void_p, src), None if dst is None else arr(ctypes.c_void_p, dst), arr(ctypes.c_int64, n), arr(ctypes.c_int32, dt), k, 0, max_norm,
                                ctypes.c_void_p(4096), nbytes, ctypes.c_void_p(64), None)

    A, B = 1 << 20, 1 << 24
    F32, F16 = _lib.GD_F32, _lib.GD_F16
    assert call([A], None, [-1], [F32]) == -1 and call([A], None, [4], [7]) == -1 and call([A + 2], None, [4], [F32]) == -1 and call([0], None, [4], [F32]) == -1
    assert call([A], [0], [4], [F32]) == -1 and call([A], [A], [4], [F32], max_norm=-1.0) == -1 and call([A], [A], [4], [F32], max_norm=math.nan) == -1
    assert call([A], None, [4], [F32], nbytes=8) == -2
    for src, dst, n, dt in (([A, A], [A, A], [4, 4], [F32, F32]),                              # the same tensor twice
                            ([A, A + 8], [A, A + 8], [4, 4], [F32, F32]),                      # two that share elements
                            ([A], [A + 4], [4], [F32]),                                        # into itself, moved
                            ([A, B], [B, A], [4, 4], [F32, F32]),                              # into each other
                            ([A, B], [A, B], [1 << 23, 4], [F16, F16])):                       # the second inside the first
        assert call(src, dst, n, dt) == -1 and b"overlaps" in lib.gd_last_error(), (src, dst)


@gpu
def test_clipping_refusals(ops):
    t = torch.ones(4, 6, device=DEV)
    bad = [lambda: ops.grad_norm([t, t.cpu()]), lambda: ops.grad_norm([t.t()]), lambda: ops.grad_norm([t[:, :3]]), lambda: ops.grad_norm([t.double()]), lambda: ops.grad_norm([t.int()]),
           lambda: ops.clip_grad_norm([t], -1.0), lambda: ops.clip_grad_norm([t], math.nan), lambda: ops.clip_grad_norm([t, t], 1.0), lambda: ops.clip_grad_norm([t, t[1:]], 1.0),
           lambda: ops.clip_grad_norm([t], 1.0, out=[]), lambda: ops.clip_grad_norm([t], 1.0, out=[t.half()]), lambda: ops.clip_grad_norm([t], 1.0, out=[t.reshape(6, 4)]),
           lambda: ops.clip_grad_norm([t[:2], t[2:]], 1.0, out=[t[1:3], torch.empty_like(t[:2])]), lambda: ops.grad_norm([t], 3)]
    for i, call in enumerate(bad):
        with pytest.raises(GeodiffError):
            call()
            pytest.fail(str(i))
    assert float(t.sum()) == 24


@gpu
def test_calls_larger_than_the_cache(ops):
    """Calls whose tensors exceed the memory-side cache store past it: the same bits as their rows give in a small call, or as torch's."""
    g = torch.Generator(device=DEV).manual_seed(8)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV).bfloat16()
    table = r(50000, 1024)
    ids = torch.randint(0, 50000, (1700, 77), generator=g, device=DEV)
    y = ops.embed_tokens(ids, table)
    assert (y.numel() + table.numel()) * 2 > 1 << 28 and bool((y == table[ids]).all())
    del y, table
    ids = torch.randint(0, 300000, (2500,), generator=g, device=DEV)
    _check_embed_bwd(ops, ids, r(2500, 512), 300000)
    x, res, gy, gs = (r(2, 20000, 1280) for _ in range(4))
    gate, pre, post = r(2, 1280), ops.Norm("layer", r(1280), r(1280)), ops.Norm("rms", r(1280))
    s, y, st = ops.block_norm(x, res, pre, post, gate, 0.5)
    d = ops.block_norm_bwd(x, res, gy, gs, st, pre, post, gate, 0.5)
    cut = lambda t: t[:, 300:420].contiguous()
    s2, y2, st2 = ops.block_norm(cut(x), cut(res), pre, post, gate, 0.5)
    d2 = ops.block_norm_bwd(cut(x), cut(res), cut(gy), cut(gs), st2, pre, post, gate, 0.5)
    assert torch.equal(cut(s), s2) and torch.equal(cut(y), y2) and torch.equal(cut(d["dx"]), d2["dx"]) and torch.equal(cut(d["dres"]), d2["dres"])
    del x, res, gy, gs, s, y, d
    grads = [r(9000, 9000), r(77), r(8191 * 8191)]
    out = [torch.zeros_like(t) for t in grads]
    n = ops.clip_grad_norm(grads, 2.0, out=out)
    total = float(_norm_ref(grads))
    assert abs(float(n) - total) <= 2 * U32 * total
    for t, o in zip(grads, out):
        _close(o, t.double() * (2.0 / (total + 1e-6)), 2, t.double().abs() * (2.0 / total))
    v = grads[0]._version
    ops.clip_grad_norm(grads, 2.0)
    assert all(torch.equal(t, o) for t, o in zip(grads, out)) and grads[0]._version > v


# ------------------------------------------------------------------------------------------------ streams, graphs
@gpu
def test_training_ops_on_another_stream_and_replayed_in_graphs(ops):
    """Every operator on a side stream, and captured: two graphs replayed in turn on new inputs, with eager work between, against the eager results."""
    g = _gen(1)
    V, C = 900, 136
    ids = torch.randint(0, V, (40, 77), generator=g).to(DEV)
    table, pos = _randn(g, V, C), _randn(g, 77, C)
    x, r, pre, po, gt, gy, gs = _block_case(ops, (4, 50, C), torch.float32, "layer", "sample", True, True, 2)
    dy = _randn(g, 40, 77, C)
    grads = [_randn(g, n) for n in (5, 9000, 70000)]
    bufs = [torch.empty_like(t) for t in grads]

    def all_ops():
        s, y, stats = ops.block_norm(x, r, pre, po, gt)
        d = ops.block_norm_bwd(x, r, gy, gs, stats, pre, po, gt)
        n = ops.clip_grad_norm(grads, 1.0, out=bufs)
        return [ops.embed_tokens(ids, table, pos), ops.embed_tokens_bwd(ids, dy, V), ops.embed_tokens_bwd(ids[:2], dy[:2], V), ops.embed_positions_bwd(dy, 80), s, y,
                *d.values(), n, *[b.clone() for b in bufs], ops.grad_norm(grads, math.inf)]

    want = all_ops()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = all_ops()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = all_ops()
        graphs.append((graph, out))
    inputs = (x, r, gy, gs, dy, table, *grads)
    for k in range(3):
        for t in inputs:
            t.copy_(_randn(g, *t.shape))
        ids.copy_(torch.randint(0, V, ids.shape, generator=g))
        want = all_ops()
        for graph, out in graphs if k % 2 else graphs[::-1]:
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want)), k
            want = all_ops()


@gpu
def test_a_captured_training_step(ops):
    """Forward, backward and clipping of embedding and block norm as one graph, replayed on new data between eager steps on leaves of their own."""
    from geodiffuser_amd import training as T
    g = _gen(21)
    V, C = 400, 72
    ids = torch.randint(0, V, (6, 77), generator=g).to(DEV)
    data = dict(table=_randn(g, V, C), pos=_randn(g, 77, C), gate=_randn(g, 6, C), g1=_randn(g, C), b1=_randn(g, C), g2=_randn(g, C), w=_randn(g, 6, 77, C))

    def step(d):
        p = {k: d[k].detach().requires_grad_() for k in ("table", "pos", "gate", "g1", "b1", "g2")}
        x = T.embed_tokens(ids, p["table"], p["pos"], 2.0)
        s, y = T.block_norm(x, x, T.Norm("layer", p["g1"], p["b1"]), post=T.Norm("rms", p["g2"]), gate=p["gate"], res_scale=0.5)
        grads = [t.contiguous() for t in torch.autograd.grad([s, y], list(p.values()), [d["w"], d["w"]])]
        return [y.detach(), ops.clip_grad_norm(grads, 3.0), *grads]

    static = {k: v.clone() for k, v in data.items()}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(static)
    for k in range(4):
        ids.copy_(torch.randint(0, V, ids.shape, generator=g))
        for t in static.values():
            t.copy_(_randn(g, *t.shape))
        want = step({k_: v.clone() for k_, v in static.items()})
        graph.replay()
        torch.cuda.synchronize()
        assert float(want[1]) > 3.0 and all(torch.equal(a, b) for a, b in zip(out, want)), k


@gpu
def test_training_ops_from_two_threads_at_once(ops):
    """Nothing is shared between calls: two threads on two streams, each over its own sizes, against the same calls one after the other."""
    import threading

    def work(seed, n, C, out):
        g = torch.Generator(device=DEV).manual_seed(seed)
        r = lambda *s: torch.randn(*s, generator=g, device=DEV)
        ids = torch.randint(0, 777, (n,), generator=g, device=DEV)
        dy, x, res, gate = r(n, C), r(3, 60, C), r(3, 60, C), r(3, C)
        norm, grads = ops.Norm("layer", r(C), r(C)), [r(k) for k in (9, 70000, 3)]
        for _ in range(20):
            s, y, st = ops.block_norm(x, res, norm, gate=gate)
            d = ops.block_norm_bwd(x, res, y, s, st, norm, gate=gate)
            buf = [torch.empty_like(t) for t in grads]
            got = [ops.embed_tokens_bwd(ids, dy, 777), ops.embed_positions_bwd(dy.view(-1, 5, C), 6), y, d["dgate"], d["dpre_gamma"], ops.clip_grad_norm(grads, 1.0, out=buf), *buf]
        out.extend(got)

    args = [(1, 5000, 64), (2, 900, 200)]
    want = [[], []]
    for a, w in zip(args, want):
        work(*a, w)
    torch.cuda.synchronize()
    got = [[], []]

    def on_stream(a, o):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            work(*a, o)
        s.synchronize()

    threads = [threading.Thread(target=on_stream, args=(a, o)) for a, o in zip(args, got)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert all(len(g_) == len(w) and all(torch.equal(a, b) for a, b in zip(g_, w)) for g_, w in zip(got, want))


@gpu
def test_training_ops_while_another_device_is_current(ops, monkeypatch):
    """A call makes its tensors' device current for its launches (here: the one there is, behind a runtime that names another)."""
    x = torch.randn(5, 64, device=DEV)
    want = ops.block_norm(x, x, ops.Norm("rms"))[1]
    seen = []
    real = torch.cuda.device
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 5)
    monkeypatch.setattr(torch.cuda, "device", lambda d: seen.append(d) or real(d))
    y = ops.block_norm(x, x, ops.Norm("rms"))[1]
    monkeypatch.undo()
    assert seen == [0] and torch.equal(y, want)


# ------------------------------------------------------------------------------------------------ as the framework uses them
@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_text_tower_embedding_keeps_its_values_and_learns(ops, dtype):
    """The tower's first layer through the operator: the bits of the unfused lookup and addition, and the gradients of table and positions."""
    from geodiffuser_amd.pipeline import TextEncoder
    torch.manual_seed(0)
    te = TextEncoder(width=64, layers=2, heads=2, vocab=500).to(DEV, dtype).eval()
    ids = torch.randint(0, 500, (3, 77), generator=_gen(2)).to(DEV)
    ids[:, 20:] = 0
    seen = []
    h = te.layers[0].register_forward_pre_hook(lambda m, a: seen.append(a[0]))
    with torch.no_grad():
        te(ids)
    te(ids)
    h.remove()
    want = te.tok(ids) + te.pos[:77]
    assert torch.equal(seen[0], want) and torch.equal(seen[1], want) and "EmbedFn" in type(seen[1].grad_fn).__name__
    gy = _randn(_gen(3), 3, 77, 64, dtype=dtype)
    dt, dp = torch.autograd.grad(seen[1], [te.tok.weight, te.pos], gy)
    ref = torch.zeros(500, 64, dtype=torch.float64, device=DEV).index_add_(0, ids.flatten(), gy.double().reshape(-1, 64))
    mag = torch.zeros_like(ref).index_add_(0, ids.flatten(), gy.double().abs().reshape(-1, 64))
    _close(dt, ref, 3 * 77, mag)
    _close(dp, gy.double().sum(0), 3, gy.double().abs().sum(0))


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_transformer_block_with_trainable_norms(ops, dtype):
    """A block whose norms learn runs them on block_norm; against the same block on stock modules in 64 bits, each gradient in relative 2-norm.
    Both round every intermediate tensor to T: about 40 such roundings lie between the loss and the first norm's gradient, each relative u in
    2-norm; 40 u bounds their sum with nothing cancelling."""
    from geodiffuser_amd import unet_sd21 as U

    class Plain:
        def __call__(self, attn, hidden_states, encoder_hidden_states=None, **kw):
            c = hidden_states if encoder_hidden_states is None else encoder_hidden_states
            return attn.to_out[0](attn.to_q(hidden_states) * torch.tanh(attn.to_k(c).mean(1, keepdim=True) + attn.to_v(c).mean(1, keepdim=True)))

    torch.manual_seed(3)
    blk = U.BasicTransformerBlock(128, 2, 64, 96).to(DEV, dtype).eval()
    for n, p in blk.named_parameters():
        p.requires_grad_("norm" in n)
        if "norm" in n:
            p.data.add_(_randn(_gen(len(n)), *p.shape, std=0.2).to(dtype))
    for a in (blk.attn1, blk.attn2):
        a.processor = Plain()
    x, ctx, w = (_randn(_gen(i), *s, dtype=dtype) for i, s in enumerate(((2, 65, 128), (2, 7, 96), (2, 65, 128))))
    calls = []
    saved = ops.block_norm
    ops.block_norm = lambda *a, **k: calls.append(1) or saved(*a, **k)
    try:
        y = blk(x, ctx)
        (y.float() * w.float()).sum().backward()
    finally:
        ops.block_norm = saved
    assert len(calls) == 3
    import copy
    ref = copy.deepcopy(blk).cpu().double()
    ref.zero_grad()
    for a in (ref.attn1, ref.attn2):
        a.processor = Plain()
    yr = ref(x.cpu().double(), ctx.cpu().double())
    (yr * w.cpu().double()).sum().backward()
    u = 40 * torch.finfo(dtype).eps / 2
    rel = lambda a, b: float((a.detach().cpu().double() - b.detach()).norm() / b.detach().norm())
    assert rel(y, yr) < u
    for (n, p), q in zip(blk.named_parameters(), ref.parameters()):
        if "norm" in n:
            assert rel(p.grad, q.grad) < u, (n, rel(p.grad, q.grad), u)
        else:
            assert p.grad is None


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_text_tower_learns_end_to_end(ops, dtype):
    """Every gradient of a two-layer tower (embedding, positions, norms on the operators; attention and projections on torch) against the same
    tower on the CPU in 64 bits, in relative 2-norm, and clipping of all of them.  Both sides round every intermediate tensor; fewer than 60
    such roundings of u relative lie on a path through two layers forward and back (bf16; each of torch's f32 products adds at most a few
    2^-24 sqrt(256) of its own, so that f32 gets 60 * 16 of them)."""
    import copy
    from geodiffuser_amd import training as T
    from geodiffuser_amd.pipeline import TextEncoder
    torch.manual_seed(5)
    te = TextEncoder(width=64, layers=2, heads=2, vocab=120, max_len=20).to(DEV, dtype)
    for n, p in te.named_parameters():
        if "ln" in n:
            p.data.add_(_randn(_gen(len(n)), *p.shape, std=0.2).to(dtype))
    ids = torch.randint(0, 120, (3, 17), generator=_gen(2))
    ids[:, 9:] = 0
    w = _randn(_gen(3), 3, 17, 64, dtype=dtype)
    calls = []
    saved = ops.block_norm, ops.embed_tokens
    ops.block_norm = lambda *a, **k: calls.append("norm") or saved[0](*a, **k)
    ops.embed_tokens = lambda *a, **k: calls.append("embed") or saved[1](*a, **k)
    try:
        y = te(ids.to(DEV))[0]
        (y.float() * w.float()).sum().backward()
    finally:
        ops.block_norm, ops.embed_tokens = saved
    assert calls == ["embed"] + ["norm"] * 4
    ref = copy.deepcopy(te).cpu().double()
    ref.zero_grad()
    yr = ref(ids)[0]
    (yr * w.cpu().double()).sum().backward()
    u = 60 * (16 * U32 if dtype == torch.float32 else torch.finfo(dtype).eps / 2)
    rel = lambda a, b: float((a.detach().cpu().double() - b.detach()).norm() / b.detach().norm())
    assert rel(y, yr) < u
    for (n, p), q in zip(te.named_parameters(), ref.parameters()):
        # (the key's bias has no gradient: softmax does not see it, so that only rounding is left there)
        a, b = (p.grad[:64], q.grad[:64]) if n.endswith("in_proj_bias") else (p.grad, q.grad)
        assert rel(a, b) < u, (n, rel(a, b), u)
    total = math.sqrt(sum(float(p.grad.double().square().sum()) for p in te.parameters()))
    norm = T.clip_grad_norm_(te.parameters(), total / 3)
    after = math.sqrt(sum(float(p.grad.double().square().sum()) for p in te.parameters()))
    assert abs(float(norm) - total) <= 2 * U32 * total and abs(after - total / 3) <= (4 * U32 + (0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2)) * total / 3


@gpu
def test_a_training_step_of_the_text_tower(ops):
    """Embedding, gated block norms and clipping as one step: every gradient against the same step on plain torch operations in 64 bits, the
    clipped norm, and a second identical step from the same state."""
    from geodiffuser_amd import training as T
    g = _gen(12)
    V, C, B, L = 300, 96, 5, 31
    ids = torch.randint(0, V, (B, L), generator=g)
    ids[:, 12:] = 0
    init = dict(table=_randn(g, V, C, std=0.5), pos=_randn(g, 77, C, std=0.2), w=_randn(g, C, C, std=C ** -0.5), gate=_randn(g, B, C), g1=_randn(g, C, mean=1.0, std=0.1),
                b1=_randn(g, C, std=0.1), g2=_randn(g, C, mean=1.0, std=0.1), g3=_randn(g, C, mean=1.0, std=0.1))
    tgt = _randn(g, B, L, C)

    def step():
        p = {k: v.clone().requires_grad_() for k, v in init.items()}
        x = T.embed_tokens(ids.to(DEV), p["table"], p["pos"], scale=C ** 0.5, padding_idx=0)
        x, h = T.block_norm(x, None, T.Norm("layer", p["g1"], p["b1"]))
        s, y = T.block_norm(h @ p["w"], x, T.Norm("rms", p["g3"]), post=T.Norm("rms", p["g2"]), gate=p["gate"], res_scale=0.5)
        loss = ((y - tgt) ** 2).mean() + 0.1 * s.square().mean()
        loss.backward()
        raw = {k: v.grad.clone() for k, v in p.items()}
        n = T.clip_grad_norm_(p.values(), 0.01)
        return loss.detach(), n, raw, {k: v.grad for k, v in p.items()}

    loss, n, raw, clipped = step()
    q = {k: v.cpu().double().requires_grad_() for k, v in init.items()}
    rms = lambda v, w: v / (v.pow(2).mean(-1, keepdim=True) + 1e-5).sqrt() * w
    x = torch.nn.functional.embedding(ids, q["table"], padding_idx=0) * C ** 0.5 + q["pos"][:L]
    h = torch.nn.functional.layer_norm(x, (C,), q["g1"], q["b1"], 1e-5)
    s = 0.5 * x + q["gate"][:, None] * rms(h @ q["w"], q["g2"])
    y = rms(s, q["g3"])
    lr = ((y - tgt.cpu().double()) ** 2).mean() + 0.1 * s.square().mean()
    lr.backward()
    # f32 throughout: 300 roundings of 2^-24 relative in 2-norm lie between any input and any gradient (sums over C and B L included)
    assert abs(float(loss) - float(lr)) <= 300 * U32 * float(lr)
    for k in q:
        assert float((raw[k].cpu().double() - q[k].grad).norm()) <= 300 * U32 * float(q[k].grad.norm()), k
    total = math.sqrt(sum(float(v.grad.square().sum()) for v in q.values()))
    assert abs(float(n) - total) <= 300 * U32 * total and total > 0.01
    f = 0.01 / (total + 1e-6)
    for k in q:
        assert float((clipped[k].cpu().double() - f * q[k].grad).norm()) <= 600 * U32 * f * float(q[k].grad.norm()), k
    again = step()
    assert torch.equal(again[1], n) and all(torch.equal(again[3][k], clipped[k]) for k in ("table", "pos", "gate", "g2", "g3"))


@gpu
def test_block_norm_autograd_without_some_gradients(ops):
    from geodiffuser_amd import training as T
    x, r, pre, po, gt, gy, gs = _block_case(ops, (2, 9, 40), torch.float32, "layer", "channel", True, True, 6)
    x.requires_grad_(), gt.requires_grad_()
    s, y = T.block_norm(x, r, pre, po, gt, 0.5)
    (dx, dg) = torch.autograd.grad(y, [x, gt], gy, retain_graph=True)               # s is not used
    v, m = _block_ref(x.detach(), r, pre, po, gt.detach(), 0.5, gy, None)
    _close(dx, v["dx"], 2 * K_ROW, m["dx"])
    _close(dg, v["dgate"], 2 * K_ROW + 18, m["dgate"])
    (dx,) = torch.autograd.grad(s, [x], gs.transpose(0, 1).contiguous().transpose(0, 1))      # y is not used; a strided incoming gradient
    v, m = _block_ref(x.detach(), r, None, po, gt.detach(), 0.5, None, gs)
    _close(dx, v["dx"], 2 * K_ROW, m["dx"])
    s, y = T.block_norm(x, None, pre)                                                # s is x: both of its uses reach it
    (dx,) = torch.autograd.grad([s, y], [x], [gs, gy])
    v, m = _block_ref(x.detach(), None, pre, None, None, 1.0, gy, gs)
    _close(dx, v["dx"], 2 * K_ROW, m["dx"])
    with torch.no_grad():
        assert not T.block_norm(x, None, pre)[1].requires_grad


@gpu
def test_clip_grad_norm_of_parameters(ops):
    from geodiffuser_amd import training as T
    m = torch.nn.Sequential(torch.nn.Linear(30, 40), torch.nn.LayerNorm(40), torch.nn.Linear(40, 3)).to(DEV)
    m[1].bias.requires_grad_(False)
    m(torch.randn(5, 30, device=DEV)).square().sum().backward()
    ref = [p.grad.clone() for p in m.parameters() if p.grad is not None]
    n = T.clip_grad_norm_(m.parameters(), 0.3)
    total = float(_norm_ref(ref))
    assert total > 0.3 and abs(float(n) - total) <= 2 * U32 * total
    for p, r in zip([p for p in m.parameters() if p.grad is not None], ref):
        want = r.double() * (0.3 / (total + 1e-6))
        _close(p.grad, want, 2, want.abs())
    assert float(T.clip_grad_norm_(torch.nn.Parameter(torch.zeros(3)), 1.0)) == 0.0


@gpu
def test_null_text_optimisation_with_clipped_gradients(ops):
    """NullInversion(max_grad_norm=...): the embedding's gradient is clipped before each Adam step.  Adam divides by the gradient's own size, so a
    clip to a size far above its epsilon changes little, and one far below it nearly stops the optimisation; without it nothing changes."""
    import cases
    from geodiffuser_amd.diffusion import load_model
    from geodiffuser_amd.inversion import NullInversion
    p, tok, sched = load_model(device="cuda:0", tiny=True, dtype=torch.float16)
    c = cases.NULL_TEXT
    traj = [torch.from_numpy(a).cuda().half() for a in cases.null_text_inputs()]

    def run(limit):
        ni = NullInversion(p, num_ddim_steps=c["steps"], device="cuda:0", guidance_scale=c["guidance"], max_grad_norm=limit)
        ni.init_prompt("")
        return torch.cat(ni.null_optimization(traj, c["inner"], c["eps"])).float() - ni.context[:1].float()

    free, loose, tight = run(None), run(1e9), run(1e-12)
    assert torch.isfinite(tight).all() and float(loose.norm()) > 0.5 * float(free.norm()) > 0
    assert float(tight.norm()) < 0.05 * float(free.norm())


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("C", [1, 2, 3, 4, 5, 7, 8, 9, 11, 15, 16, 17, 31, 33, 63, 65, 129, 513, 514, 517, 1023, 1027, 4097])
def test_rows_of_every_width_stay_in_their_place(ops, monkeypatch, dtype, C):
    """Every result lies inside a larger buffer, at an address that is a multiple of the element only: nothing around it is written, and the
    results are those of the ordinary call."""
    g = _gen(C)
    V, B, L, P = 23, 5, 4, 7
    ids, table, pos, dy = torch.randint(0, V, (B, L), generator=g).to(DEV), _randn(g, V, C, dtype=dtype), _randn(g, P, C, dtype=dtype), _randn(g, B, L, C, dtype=dtype)
    many, dmany = torch.randint(0, V, (1100,), generator=g).to(DEV), _randn(g, 1100, C, dtype=dtype)
    x, res, gy, gs = (_randn(g, B, L, C, dtype=dtype) for _ in range(4))
    pre, post = (ops.Norm(k, _randn(g, C, dtype=dtype), _randn(g, C, dtype=dtype), 1e-5) for k in ("layer", "rms"))
    gate = _randn(g, B, C, dtype=dtype)

    def results():
        s, y, stats = ops.block_norm(x, res, pre, post=post, gate=gate)
        d = ops.block_norm_bwd(x, res, gy, gs, stats, pre, post=post, gate=gate)
        return [ops.embed_tokens(ids, table, pos), ops.embed_tokens_bwd(ids, dy, V), ops.embed_tokens_bwd(many, dmany, V), ops.embed_positions_bwd(dy, P), s, y, stats,
                *(d[k] for k in sorted(d))]
    plain = results()
    empty, like, around = torch.empty, torch.empty_like, []

    def inside(*shape, dtype=torch.float32, device=None):
        shape = torch.Size(shape[0] if len(shape) == 1 and not isinstance(shape[0], int) else shape)
        front, n = 64 if dtype == torch.uint8 else 33, shape.numel()          # (workspaces keep their alignment)
        buf = empty(front + n + 40, dtype=dtype, device=device).fill_(7)
        around.extend((buf[:front], buf[front + n:]))
        return buf[front:front + n].view(shape)
    monkeypatch.setattr(torch, "empty", inside)
    monkeypatch.setattr(torch, "empty_like", lambda t: inside(*t.shape, dtype=t.dtype, device=t.device))
    moved = results()
    monkeypatch.undo()
    assert torch.empty is empty and torch.empty_like is like and len(around) >= 2 * len(plain)
    assert all(bool((a == 7).all()) for a in around)
    fi = torch.finfo(dtype)
    for a, b in zip(plain, moved):
        # (the column sums and row sums may be dealt out otherwise; values of ~1 and sums of at most 1100 of them)
        assert a.shape == b.shape and bool(((a.double() - b.double()).abs() <= fi.eps * b.double().abs() + 1100 * 64 * U32 * 8 + fi.smallest_normal).all())


@gpu
@pytest.mark.parametrize("n,V", [(1025, 1), (1025, 255), (1025, 256), (1025, 257), (4096, (1 << 20) - 1), (8192, 1 << 19), (8192, (1 << 19) + 1), (8193, 5000), (16384, 1 << 18), (16384, 300), (16385, 300)])
@pytest.mark.parametrize("wide", [False, True])
def test_embedding_gradient_at_the_borders_of_its_sorts(ops, n, V, wide):
    """Sizes beside each choice of sort, 32- and 64-bit ids; frequent tokens, all of one block of 256, ids outside the table and a padding row."""
    g = _gen(n + V)
    dy = _randn(g, n, 3)
    for kind in range(4):
        ids = (V * torch.rand(n, generator=g, dtype=torch.float64) ** (1, 6, 1, 1)[kind]).long().clamp(0, V - 1)
        if kind == 1:
            ids[torch.rand(n, generator=g) < 0.5] = V // 2
        elif kind == 2:
            ids = V - 1 - ids % min(V, 200)
        elif kind == 3:
            ids[::3] = torch.tensor([-1, V, -(1 << 31), (1 << 31) - 1])[torch.arange(0, n, 3) // 3 % 4]
        _check_embed_bwd(ops, (ids if wide else ids.int()).to(DEV), dy, V, scale=0.5, padding_idx=None if kind == 0 else V // 2)


@gpu
def test_sizes_beyond_32_bits_are_refused(ops):
    """Widths and row counts that the library takes as 32-bit numbers: 2^32 + 8 channels must not be taken for 8."""
    big = torch.empty((1 << 32) + 8, dtype=torch.float16, device=DEV)
    one, ids = big.view(1, -1), torch.zeros(1, dtype=torch.long, device=DEV)
    few = torch.zeros(1, 1, 1, dtype=torch.float16, device=DEV)
    for call in (lambda: ops.block_norm(one, None, ops.Norm("layer")), lambda: ops.block_norm_bwd(one, None, one, None, torch.zeros(1, 4, device=DEV), ops.Norm("layer")),
                 lambda: ops.embed_tokens(ids, one), lambda: ops.embed_tokens_bwd(ids, one, 1), lambda: ops.embed_positions_bwd(big.view(1, -1, 1), (1 << 32) + 8),
                 lambda: ops.embed_positions_bwd(big.view(1, 1, -1), 1), lambda: ops.embed_positions_bwd(few, (1 << 32) + 8)):
        with pytest.raises(GeodiffError, match="at most"):
            call()


@gpu
def test_launches_of_more_than_2_32_threads(ops):
    """A launch has fewer than 2^32 threads along an axis: 2^26 rows of a wave each, and 2^29 of eight lanes, reach that."""
    R = (1 << 26) + 5
    g = _gen(3)
    x = torch.zeros(R, 8, dtype=torch.float16, device=DEV)
    x[-9:] = x[:9] = tail = _randn(g, 9, 8, dtype=torch.float16)
    n = ops.Norm("layer", _randn(g, 8, dtype=torch.float16), None)
    _, y, st = ops.block_norm(x, None, n)
    _, y2, st2 = ops.block_norm(tail, None, n)
    for at in (slice(0, 9), slice(R - 9, R)):
        assert torch.equal(y[at], y2) and torch.equal(st[at], st2)
    assert not bool(y[9:-9].any())
    dx = ops.block_norm_bwd(x, None, x, None, st, n, need=["dx"])["dx"]
    assert torch.equal(dx[-9:], ops.block_norm_bwd(tail, None, tail, None, st2, n, need=["dx"])["dx"])
    del x, y, st, dx
    N = (1 << 29) + 3
    table = _randn(g, 5, 7, dtype=torch.float16)
    ids = torch.zeros(N, dtype=torch.int32, device=DEV)
    ids[-1], ids[-2], ids[1] = 4, 3, 2
    y = ops.embed_tokens(ids, table)
    assert torch.equal(y[-2:], table[[3, 4]]) and torch.equal(y[:2], table[[0, 2]])
    del ids
    for part in y[2:-2].split(1 << 26):
        assert bool((part == table[0]).all())
    del y, part
    V = (1 << 30) + 7                                        # zero rows: 2^22 workgroups of 1024 threads and more
    torch.full((V, 1), 7.0, dtype=torch.float16, device=DEV)  # (what the gradient's memory holds before)
    d = ops.embed_tokens_bwd(torch.tensor([V - 1, 3, V - 1], device=DEV), torch.ones(3, 1, dtype=torch.float16, device=DEV), V)
    assert float(d[-1]) == 2.0 and float(d[3]) == 1.0 and int((d != 0).sum()) == 2
    P = (1 << 31) - 1                                        # position rows: 6 billion single elements, summed by one workgroup a column and by several
    for B in (1, 100):
        torch.full((P, 3), 7.0, dtype=torch.float16, device=DEV)
        d = ops.embed_positions_bwd(torch.ones(B, 2, 3, dtype=torch.float16, device=DEV), P)
        assert bool((d[:2] == B).all()) and int((d[2:] != 0).sum()) == 0


def test_gradient_launches_beyond_2_32_threads_are_refused():
    """(on the host, with addresses that are never followed) 2^30 - 1 positions need 2^24 workgroups of 256 threads for the joins."""
    from geodiffuser_amd import _lib
    lib = _lib.load()
    A, n = 1 << 20, (1 << 30) - 1
    assert lib.gd_embed_bwd(ctypes.c_void_p(A), 1, n, ctypes.c_void_p(A), 100, 1, -1, 1.0, ctypes.c_void_p(A), ctypes.c_void_p(A), lib.gd_embed_bwd_workspace_bytes(n, 100, 1), 2, None) == -4


def test_block_norm_refuses_parameters_of_a_norm_that_is_not_there():
    """(on the host, with addresses that are never followed) the forward would leave them out and the backward apply them."""
    from geodiffuser_amd import _lib
    lib = _lib.load()
    A = 1 << 20
    ok = dict(x=A, res=A, gate=A, y=A, s=A, stats=A, rows=8, rows_per_gate=8, gate_ld=64, C=64, pre_kind=1, res_scale=1.0)
    for bad in (dict(post_gamma=A), dict(post_beta=A), dict(pre_kind=0, y=0, pre_gamma=A), dict(pre_kind=0, y=0, pre_beta=A)):
        f = _lib.GdBlockNorm(**{**ok, **bad})
        assert lib.gd_block_norm(ctypes.byref(f), 2, None) == -1, bad
        assert lib.gd_block_norm_bwd(ctypes.byref(_lib.GdBlockNormBwd(f=f, gs=A, dx=A)), None, 0, 2, None) == -1, bad


class _NoAttention(torch.nn.Module):
    """Stands where a text layer has its attention: one product, which every transform of torch can follow."""

    def __init__(self, d):
        super().__init__()
        self.lin = torch.nn.Linear(d, d)

    def forward(self, q, k, v, attn_mask=None, need_weights=False):
        return torch.tanh(self.lin(q)), None


def _small_tower(dev, dtype=torch.float32):
    from geodiffuser_amd.pipeline import TextEncoder
    torch.manual_seed(7)
    te = TextEncoder(width=32, layers=1, heads=2, vocab=50, max_len=12)
    te.layers[0].attn = _NoAttention(32)
    return te.to(dev, dtype)


def _tower_views(te, ids):
    """What torch's transforms say of the tower: name -> a list of tensors."""
    from torch.autograd import forward_ad
    from torch._subclasses.fake_tensor import FakeTensorMode
    params = {k: p.detach() for k, p in te.named_parameters()}
    call = lambda p, i: torch.func.functional_call(te, p, (i,))[0]
    loss = lambda p, i: call(p, i).square().sum()
    t = {k: torch.sin(torch.arange(p.numel(), device=p.device, dtype=p.dtype)).view(p.shape) for k, p in params.items()}

    def dual():
        with forward_ad.dual_level():
            return [forward_ad.unpack_dual(call({k: forward_ad.make_dual(p, t[k]) for k, p in params.items()}, ids)).tangent.clone()]

    def fake():
        with FakeTensorMode(allow_non_fake_inputs=True) as mode:
            y = te(mode.from_tensor(ids))[0]
        assert type(y).__name__ == "FakeTensor"
        return [torch.zeros(y.shape)]

    def second(keys=("tok.weight", "pos", "layers.0.ln1.weight", "ln_f.bias", "layers.0.fc1.weight")):
        """gradient of the gradient's inner product with t"""
        p = {k: v.clone().requires_grad_() for k, v in params.items()}
        g = torch.autograd.grad(loss(p, ids), [p[k] for k in keys], create_graph=True)
        return list(torch.autograd.grad(sum((a * t[k]).sum() for a, k in zip(g, keys)), [p[k] for k in keys]))

    def batched():
        p = {k: v.clone().requires_grad_() for k, v in params.items()}
        y = call(p, ids)
        return list(torch.autograd.grad(y, list(p.values()), torch.stack([y.detach().cos(), y.detach().sin()]), is_grads_batched=True))

    return {
        "grad": lambda: list(torch.func.grad(loss)(params, ids).values()),
        "vmap": lambda: [torch.func.vmap(call, in_dims=(None, 0))(params, ids[:, None])],
        "vmap of grad": lambda: list(torch.func.vmap(torch.func.grad(loss), in_dims=(None, 0))(params, ids[:, None]).values()),
        "jvp": lambda: [torch.func.jvp(lambda p: call(p, ids), (params,), (t,))[1]],
        "dual": dual, "fake": fake, "second": second, "batched": batched,
        "traced": lambda: [torch.jit.trace(te, (ids,), strict=False, check_trace=False)(ids.flip(0))[0]],
        "compiled": lambda: [torch.compile(te, backend="eager", fullgraph=True)(ids)[0]],
    }


_VIEWS = ["grad", "vmap", "vmap of grad", "jvp", "dual", "fake", "second", "batched", "traced", "compiled"]


@gpu
@pytest.mark.parametrize("view", _VIEWS)
def test_text_tower_under_transforms(ops, view):
    """torch's transforms reach through the tower on the GPU as they do on the CPU in 64 bits.  f32: fewer than 60 roundings lie on a path forward
    and back, each product adding at most a few 2^-24 sqrt(32), and as many again for a second derivative: 60 * 16 * 2 of 2^-24 in relative
    2-norm, over all results of a view together."""
    torch._dynamo.reset()
    ids = torch.randint(0, 50, (3, 9), generator=_gen(2))
    ids[:, 5:] = 0
    te = _small_tower(DEV)
    got = _tower_views(te, ids.to(DEV))[view]()
    want = _tower_views(_small_tower("cpu").double(), ids)[view]()
    assert len(got) == len(want) and all(a.shape == b.shape for a, b in zip(got, want))
    flat = lambda ts: torch.cat([t.detach().cpu().double().flatten() for t in ts])
    a, b = flat(got), flat(want)
    assert float((a - b).norm()) <= 2 * 60 * 16 * U32 * float(b.norm())


def test_what_is_taken_for_an_ordinary_pass():
    from torch.autograd import forward_ad
    from torch._subclasses.fake_tensor import FakeTensorMode
    from geodiffuser_amd import training as T
    x, p = torch.ones(3), torch.nn.Parameter(torch.ones(3))
    seen = []
    look = lambda t: seen.append(T.in_plain_torch(t)) or t.sum()
    assert T.in_plain_torch(x, p) and T.in_plain_torch()
    with torch.no_grad(), torch.device("cpu"):
        assert T.in_plain_torch(x)
    torch.func.grad(look)(x), torch.func.vmap(look)(x), torch.func.jvp(look, (x,), (x,)), torch.jit.trace(look, (x,), check_trace=False)
    with forward_ad.dual_level():
        look(forward_ad.make_dual(x, x))
    with FakeTensorMode() as mode:
        look(mode.from_tensor(x))
    fake = mode.from_tensor(x)

    class Sub(torch.Tensor):
        pass
    seen += [T.in_plain_torch(x, fake), T.in_plain_torch(x.as_subclass(Sub))]
    assert len(seen) == 8 and not any(seen) and T.in_plain_torch(x)
    ln = torch.nn.LayerNorm(3)
    assert T.is_stock(ln, torch.nn.LayerNorm) and not T.is_stock(ln, torch.nn.Embedding)
    h = torch.nn.modules.module.register_module_forward_hook(lambda *a: None)
    assert not T.is_stock(ln, torch.nn.LayerNorm)
    h.remove()
    for register in (ln.register_forward_hook, ln.register_forward_pre_hook, ln.register_full_backward_hook):
        h = register(lambda *a: None)
        assert not T.is_stock(ln, torch.nn.LayerNorm)
        h.remove()
    assert T.is_stock(ln, torch.nn.LayerNorm)
    ln.forward = lambda t: t
    assert not T.is_stock(ln, torch.nn.LayerNorm)


def _gradients_case(kind, gate, post, res, given, dtype=torch.float64):
    g = _gen(len(kind) + 3 * res)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64).to(dtype).requires_grad_()
    t = dict(x=r(2, 3, 5), res=r(2, 3, 5) if res else None, gate=None if gate is None else r(5) if gate == "channel" else r(2, 5))
    for k in ("pre", "post"):
        there = k == "pre" or post
        t[k + "_gamma"], t[k + "_beta"] = (r(5), r(5)) if there else (None, None)
    return t, r(2, 3, 5) if "y" in given else None, r(2, 3, 5) if "s" in given else None


@pytest.mark.parametrize("given", ["ys", "y", "s"])
@pytest.mark.parametrize("kind,gate,post,res", [("layer", None, None, False), ("layer", "sample", "rms", True), ("rms", "channel", "layer", True), ("rms", "sample", None, False)])
def test_block_norm_gradients_in_torch(kind, gate, post, res, given):
    """The form that higher derivatives take, in 64 bits: equal to autograd of the definition (fewer than 200 roundings of 2^-53 of values
    below 100), and differentiable itself."""
    from geodiffuser_amd import training as T
    t, gy, gs = _gradients_case(kind, gate, post, res, given)
    names = {"d" + k: v for k, v in t.items() if v is not None}

    def norm(v, kind, gamma, beta):
        c = v - v.mean(-1, keepdim=True) if kind == "layer" else v
        return c / (c.square().mean(-1, keepdim=True) + EPS).sqrt() * gamma + beta

    h = t["x"] if post is None else norm(t["x"], post, t["post_gamma"], t["post_beta"])
    h = h if gate is None else h * (t["gate"] if gate == "channel" else t["gate"][:, None])
    s = h + 0.5 * t["res"] if res else h
    y = norm(s, kind, t["pre_gamma"], t["pre_beta"])
    outs = [(o, g) for o, g in ((y, gy), (s, gs)) if g is not None]
    want = torch.autograd.grad([o for o, _ in outs], list(names.values()), [g for _, g in outs], allow_unused=True)

    def grads(*leaves):
        p = dict(zip(names, leaves))
        pre = T.Norm(kind, p["dpre_gamma"], p["dpre_beta"], EPS)
        po = T.Norm(post, p["dpost_gamma"], p["dpost_beta"], EPS) if post else None
        d = T._block_norm_grads_in_torch(p["dx"], p.get("dres"), leaves[len(names)] if gy is not None else None, leaves[-1] if gs is not None else None, pre, po, p.get("dgate"), 0.5)
        return tuple(d[k] for k in names)
    leaves = list(names.values()) + [g for g in (gy, gs) if g is not None]
    for k, a, b in zip(names, grads(*leaves), want):
        assert a.shape == names[k].shape and float((a - (0 if b is None else b)).abs().max()) < 200 * 2.0 ** -53 * 100, k
    assert torch.autograd.gradcheck(lambda *a: tuple(v for v in grads(*a) if v.requires_grad), leaves)


def test_embedding_gradients_in_torch():
    from geodiffuser_amd import training as T
    ids = torch.tensor([[0, 3, -1, 2], [3, 9, 2, 2 ** 40]])
    dy = torch.randn(2, 4, 3, generator=_gen(1), dtype=torch.float64, requires_grad=True)
    for i in (ids, ids.clamp(max=9).int()):
        table, pos = T._embed_grads_in_torch(i, dy, 5, 6, 0.5, 2)
        want = torch.zeros(5, 3, dtype=torch.float64)
        want[0], want[3] = 0.5 * dy[0, 0], 0.5 * (dy[0, 1] + dy[1, 0])
        assert torch.allclose(table, want, rtol=0, atol=1e-15) and torch.equal(pos, torch.cat([dy.sum(0), torch.zeros(2, 3, dtype=torch.float64)]))
        assert torch.autograd.gradcheck(lambda d: T._embed_grads_in_torch(i, d, 5, 6, 0.5, 2), (dy,))
    assert T._embed_grads_in_torch(ids[0], dy[0], 0, None, 1.0, None)[0].shape == (0, 3) and T._embed_grads_in_torch(ids[:0], dy[:0], 4, 4, 1.0, None)[1].sum() == 0


@gpu
def test_second_derivatives_of_the_training_operators(ops):
    """Embedding, then a gated block norm with both norms: second derivatives against the same in 64 bits on the CPU.  f32: 2 * 400 roundings of
    2^-24 in relative 2-norm for all of them together."""
    from geodiffuser_amd import training as T
    g = _gen(31)
    ids = torch.randint(0, 20, (3, 6), generator=g)
    init = dict(table=_randn(g, 20, 24, dev="cpu"), pos=_randn(g, 6, 24, dev="cpu"), gate=_randn(g, 3, 24, dev="cpu"), g1=_randn(g, 24, dev="cpu"), b1=_randn(g, 24, dev="cpu"),
                g2=_randn(g, 24, dev="cpu"), w=_randn(g, 24, 24, dev="cpu"))
    t = {k: _randn(g, *v.shape, dev="cpu") for k, v in init.items()}

    def norm(v, kind, gamma, beta=0.0):
        c = v - v.mean(-1, keepdim=True) if kind == "layer" else v
        return c / (c.square().mean(-1, keepdim=True) + EPS).sqrt() * gamma + beta

    def second(dev, dtype):
        p = {k: v.to(dev, dtype).requires_grad_() for k, v in init.items()}
        if dev == "cpu":
            x = 2.0 * torch.nn.functional.embedding(ids, p["table"]) + p["pos"]
            s = 0.5 * x + p["gate"][:, None] * norm(x @ p["w"], "rms", p["g2"])
            y = norm(s, "layer", p["g1"], p["b1"])
        else:
            x = T.embed_tokens(ids.to(dev), p["table"], p["pos"], 2.0)
            s, y = T.block_norm(x @ p["w"], x, T.Norm("layer", p["g1"], p["b1"], EPS), post=T.Norm("rms", p["g2"], None, EPS), gate=p["gate"], res_scale=0.5)
        first = torch.autograd.grad(y.pow(3).mean() + s.square().mean(), list(p.values()), create_graph=True)
        z = sum((a * t[k].to(dev, dtype)).sum() for a, k in zip(first, p))
        return torch.cat([a.detach().cpu().double().flatten() for a in (*first, *torch.autograd.grad(z, list(p.values())))])
    got, want = second(DEV, torch.float32), second("cpu", torch.float64)
    assert float((got - want).norm()) <= 2 * 400 * U32 * float(want.norm())


@gpu
def test_clip_grad_norm_of_gradients_in_any_dense_order(ops):
    """Parameters whose axes lie in another order have gradients that do too: the norm and every value as torch's function has them."""
    from geodiffuser_amd import training as T
    for kind in (2.0, math.inf):
        g = _gen(4)
        flat = _randn(g, 6000)
        params = [torch.nn.Parameter(p) for p in (
            _randn(g, 40, 65).t(), _randn(g, 4, 3, 5, 7, 6).to(memory_format=torch.channels_last_3d), _randn(g, 5, 6, 7).permute(2, 0, 1), _randn(g, 9, 2, 4).transpose(0, 1),
            flat[1001:1001 + 24].view(4, 6).t(), _randn(g, 1, 7, dtype=torch.bfloat16).t(), _randn(g, 8, 6, dtype=torch.float16).t(), _randn(g, 33))]
        sum((p.float() * p.float().sin()).sum() for p in params).backward()
        assert sum(not p.grad.is_contiguous() for p in params) >= 6
        ref, versions = [p.grad.clone() for p in params], [p.grad._version for p in params]
        total = float(_norm_ref(ref, kind))
        n = T.clip_grad_norm_(params, total / 7, kind)
        assert abs(float(n) - total) <= 2 * U32 * total
        for p, r, v in zip(params, ref, versions):
            assert p.grad.stride() == r.stride() and p.grad._version > v
            want = r.double() * (total / 7 / (total + 1e-6))
            _close(p.grad, want, 4, want.abs())                               # the norm to f32 in the test's factor, the factor, the product
    p = torch.nn.Parameter(torch.ones(4, 6, device=DEV))
    p.grad = torch.ones(8, 6, device=DEV)[::2]                                # gaps: not dense
    with pytest.raises(GeodiffError, match="contiguous"):
        T.clip_grad_norm_(p, 1.0)
    p.grad = torch.ones(4, 1, device=DEV).expand(4, 6)
    with pytest.raises(GeodiffError, match="contiguous"):
        T.clip_grad_norm_(p, 1.0)
    p.grad = torch.ones(4, 6, device=DEV)
    with pytest.raises(GeodiffError, match="overlaps"):
        T.clip_grad_norm_([p, p], 1.0)
    p.grad = None
    assert T.clip_grad_norm_([p], 1.0).device == p.device and float(T.clip_grad_norm_([], 1.0)) == 0.0


@gpu
def test_refused_clipping_leaves_its_tensors_as_they_were(ops):
    """A call that the library refuses has written nothing, and autograd is not told otherwise."""
    t, o = torch.ones(6, device=DEV), torch.ones(6, device=DEV)
    for call in (lambda: ops.clip_grad_norm([t, t], 1.0), lambda: ops.clip_grad_norm([t, o], 1.0, out=[o, torch.empty_like(t)])):
        v = t._version, o._version
        with pytest.raises(GeodiffError, match="overlaps"):
            call()
        assert (t._version, o._version) == v and bool((t == 1).all())
    v = t._version, o._version
    ops.clip_grad_norm([t], 1.0, out=[o])
    assert t._version == v[0] and o._version > v[1]
    ops.clip_grad_norm([t], 1.0)
    assert t._version > v[0]


@gpu
def test_text_tower_takes_a_batch_of_prompts_only(ops):
    """Ids without a batch axis end where the unfused addition ends them, on the GPU as on the CPU."""
    for dev in ("cpu", DEV):
        te = _small_tower(dev)
        with pytest.raises(IndexError):
            te(torch.zeros(32, dtype=torch.long, device=dev))


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("C", [1, 5, 8, 24, 65, 333, 513, 1027, 2056, 4097])
def test_results_do_not_depend_on_where_they_lie(ops, monkeypatch, dtype, C):
    """Outputs at an address that is a multiple of the element only, and inputs there: the embeddings' bits are those of the ordinary call, the
    norms' results as near to the 64-bit ones as any."""
    g = _gen(C)
    V, B, L, P = 23, 5, 4, 7
    ids, table, pos, dy = torch.randint(0, V, (B, L), generator=g).to(DEV), _randn(g, V, C, dtype=dtype), _randn(g, P, C, dtype=dtype), _randn(g, B, L, C, dtype=dtype)
    many, dmany = torch.randint(0, V, (1100,), generator=g).to(DEV), _randn(g, 1100, C, dtype=dtype)
    dbatch = _randn(g, 130, L, C, dtype=dtype)
    embed = lambda mis: [ops.embed_tokens(ids, mis(table), mis(pos), 3.0), ops.embed_tokens_bwd(ids, mis(dy), V), ops.embed_tokens_bwd(many, mis(dmany), V),
                         ops.embed_positions_bwd(mis(dy), P), ops.embed_positions_bwd(mis(dbatch), P)]
    x, r, pre, po, gt, gy, gs = _block_case(ops, (B, L, C), dtype, "layer", "sample", True, True, C)

    def norms(mis):
        n, p = (ops.Norm(t.kind, mis(t.gamma), mis(t.beta), t.eps) for t in (pre, po))
        s, y, stats = ops.block_norm(mis(x), mis(r), n, p, mis(gt), 0.5)
        return {"s": s, "y": y, **ops.block_norm_bwd(mis(x), mis(r), mis(gy), mis(gs), stats, n, p, mis(gt), 0.5)}
    same = lambda t: t
    want, (v, m) = embed(same), _block_ref(x, r, pre, po, gt, 0.5, gy, gs)
    moved_inputs = embed(_misaligned), norms(_misaligned)
    empty = torch.empty

    def inside(*shape, dtype=torch.float32, device=None):
        shape = torch.Size(shape[0] if len(shape) == 1 and not isinstance(shape[0], int) else shape)
        front = 64 if dtype == torch.uint8 else 33                               # (workspaces keep their alignment)
        return empty(front + shape.numel(), dtype=dtype, device=device)[front:].view(shape)
    monkeypatch.setattr(torch, "empty", inside)
    monkeypatch.setattr(torch, "empty_like", lambda t: inside(*t.shape, dtype=t.dtype, device=t.device))
    moved_outputs = embed(same), norms(same)
    monkeypatch.undo()
    for e, n in (moved_inputs, moved_outputs):
        assert all(torch.equal(a, b) for a, b in zip(e, want))
        for k, t in n.items():
            _close(t, v[k], (1 if k in ("s", "y") else 2) * K_ROW + (B * L if k[1:] in ("gate", "pre_gamma", "pre_beta", "post_gamma", "post_beta") else 0), m[k], k)


@gpu
@pytest.mark.parametrize("n,V", [((1 << 20) + 1, 300), (1400000, 50000), (1300000, 100001)])
def test_embedding_gradient_of_more_positions_than_a_sort_keeps_in_registers(ops, n, V):
    """More than 2048 positions a workgroup of the sort, two and three passes of it, half of them one token.  Whole numbers up to 8 as gradients: sums
    of a million of them are exact in 32 bits in any order, and a position at a wrong place shows."""
    g = torch.Generator(device=DEV).manual_seed(n)
    ids = torch.randint(0, V, (n,), generator=g, device=DEV)
    ids[torch.rand(n, generator=g, device=DEV) < 0.5] = V // 3
    dy = torch.randint(-8, 9, (n, 5), generator=g, device=DEV).float()
    ref = torch.stack([torch.bincount(ids.cpu(), weights=col.double(), minlength=V) for col in dy.cpu().t()], 1).to(DEV)
    for i in (ids, ids.int()):
        assert torch.equal(ops.embed_tokens_bwd(i, dy, V).double(), ref)
    ref[V // 3] = 0
    assert torch.equal(ops.embed_tokens_bwd(ids, dy, V, padding_idx=V // 3).double(), ref)


@gpu
def test_null_text_optimiser_sees_clipped_gradients(ops, monkeypatch):
    """What Adam is handed in NullInversion(max_grad_norm=...): gradients of that norm where they were longer, the gradients themselves where
    not.  f32 or f16 gradients: the clipped norm is off by the factor's and each element's rounding, at most (2 2^-24 + u) of it."""
    import cases
    from geodiffuser_amd import inversion, training as T
    from geodiffuser_amd.diffusion import load_model
    p, tok, sched = load_model(device="cuda:0", tiny=True, dtype=torch.float16)
    c = cases.NULL_TEXT
    traj = [torch.from_numpy(a).cuda().half() for a in cases.null_text_inputs()]
    before, after = [], []
    real, step = T.clip_grad_norm_, torch.optim.Adam.step

    def clip(ps, limit):
        grad = ps.grad.clone()
        n = real(ps, limit)
        before.append((float(n), float(grad.double().norm()), grad))
        return n

    def look(self, *a, **k):
        after.append(self.param_groups[0]["params"][0].grad.clone())
        return step(self, *a, **k)
    monkeypatch.setattr(T, "clip_grad_norm_", clip)
    monkeypatch.setattr(torch.optim.Adam, "step", look)

    def run(limit):
        before.clear(), after.clear()
        ni = inversion.NullInversion(p, num_ddim_steps=c["steps"], device="cuda:0", guidance_scale=c["guidance"], max_grad_norm=limit)
        ni.init_prompt("")
        ni.null_optimization(traj, c["inner"], c["eps"])
        assert after and (limit is None or len(before) == len(after))

    run(None)
    assert not before
    first = float(after[0].double().norm())
    run(1e9)
    assert first > 0 and all(torch.equal(g, a) and abs(n - e) <= 2 * U32 * e for (n, e, g), a in zip(before, after))
    limit = first / 4
    run(limit)
    u = 0.0 if after[0].dtype == torch.float32 else torch.finfo(after[0].dtype).eps / 2
    assert before[0][0] > limit
    for (n, e, g), a in zip(before, after):
        assert abs(float(a.double().norm()) - min(e, limit)) <= (4 * U32 + u) * limit + 1e-6


@pytest.mark.parametrize("dev", ["cpu", pytest.param(DEV, marks=gpu)])
def test_text_tower_is_scriptable(dev):
    """torch.jit.script compiles the tower (its plain operations) and gives its values; f32: the 60 * 16 roundings of a pass."""
    te = _small_tower(dev).eval()
    te.layers[0].attn = torch.nn.MultiheadAttention(32, 2, batch_first=True).to(dev).eval()
    ids = torch.randint(0, 50, (2, 9), generator=_gen(1)).to(dev)
    got, want = torch.jit.script(te)(ids)[0], te(ids)[0]
    assert float((got - want).norm()) <= 60 * 16 * U32 * float(want.norm())
