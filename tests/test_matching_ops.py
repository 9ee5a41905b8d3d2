"""Cross attention, rotary positions and the RMS norm against their plain 64-bit forms, their
refusals, and a matching layer made of them.  Tolerances: oracle/matching_oracle.py derives them."""
import ctypes
import math

import pytest
import torch

from oracle import matching_oracle as O
from realtime_stereo_matcher_amd import _lib, functional as F

gpu = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def name(dtype):
    return str(dtype).replace("torch.", "")


def normal(gen, *shape, dtype=torch.float32, scale=1.0):
    """Values that the type holds exactly, made on the host from the generator alone."""
    return (torch.randn(shape, generator=gen) * scale).to(dtype)


def near(got, want, tol, what):
    got = got.detach().cpu().double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    same = (got == want) | (got.isnan() & want.isnan())
    off = torch.where(same, 0.0, (got - want).abs())
    over = ~(off <= tol)
    assert not bool(over.any()), (
        f"{what}: {int(over.sum())} of {over.numel()} values off, worst by "
        f"{float((off / tol.clamp_min(1e-300)).nan_to_num(nan=math.inf).max()):.3g} of the bound, first at "
        f"{over.nonzero()[0].tolist()}")


# --------------------------------------------------------------------------------- the plain forms
def test_oracle_attention_gradients_are_differences():
    """The oracle's gradients against central differences of its output (64 bits: h^2 = 1e-10)."""
    gen = torch.Generator().manual_seed(1)
    q, k, v, g = (torch.randn(s, generator=gen, dtype=torch.float64)
                  for s in ((2, 5, 4, 8), (2, 7, 2, 8), (2, 7, 2, 8), (2, 5, 4, 8)))
    ok = O.allowed(2, 5, 7, band=4, lengths=torch.tensor([7, 3]))

    def out(q, k, v):
        return (O.attention(q.float().double(), k, v, 0.4, ok)[0]["out"] * g).sum()

    # the oracle rounds nothing: pass 64-bit tensors straight through
    val, _ = O.attention(q, k, v, 0.4, ok, g)
    h = 1e-5
    for x, grad in ((q, val["dq"]), (k, val["dk"]), (v, val["dv"])):
        d = torch.randn(x.shape, generator=gen, dtype=torch.float64)
        parts = [(q + e * d if x is q else q, k + e * d if x is k else k, v + e * d if x is v else v)
                 for e in (h, -h)]
        diff = [(O.attention(*p, 0.4, ok)[0]["out"] * g).sum() for p in parts]
        assert abs((diff[0] - diff[1]) / (2 * h) - (grad * d).sum()) < 1e-7


def test_oracle_norm_gradients_are_differences():
    gen = torch.Generator().manual_seed(2)
    x, r, w, g, z = (torch.randn(s, generator=gen, dtype=torch.float64)
                     for s in ((3, 7), (3, 7), (7,), (3, 7), (3, 7)))
    val, _ = O.rms_norm(x, w, r, 1e-3, g, z)

    def f(x, w):
        o, _ = O.rms_norm(x, w, r, 1e-3)
        return (o["y"] * g).sum() + (o["summed"] * z).sum()

    h = 1e-5
    d = torch.randn(x.shape, generator=gen, dtype=torch.float64)
    assert abs((f(x + h * d, w) - f(x - h * d, w)) / (2 * h) - (val["dx"] * d).sum()) < 1e-7
    d = torch.randn(w.shape, generator=gen, dtype=torch.float64)
    assert abs((f(x, w + h * d) - f(x, w - h * d)) / (2 * h) - (val["dweight"] * d).sum()) < 1e-7


def test_rotary_frequencies():
    f = F.rotary_frequencies(8)
    assert f.dtype == torch.float64
    assert torch.allclose(f, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64), rtol=1e-14)
    assert torch.equal(F.rotary_frequencies(8, scaling="linear", factor=4.0), f / 4)
    b = F.rotary_frequencies(8, scaling="base", factor=4.0)
    assert b[0] == 1.0 and abs(b[3] / f[3] - 0.25) < 1e-14
    p = F.rotary_frequencies(8, scaling="parts", factor=4.0, original_length=1000, low=1.0, high=32.0)
    turns = 1000 * f / (2 * math.pi)  # 159, 15.9, 1.59, 0.159
    keep = ((turns - 1) / 31).clamp(0, 1)
    assert p[0] == f[0] and p[3] == f[3] / 4
    assert torch.allclose(p, f * keep + f / 4 * (1 - keep), rtol=1e-14)
    for bad in (dict(dim=7), dict(dim=0), dict(dim=8, base=0.0), dict(dim=8, factor=-1.0),
                dict(dim=8, scaling="what"), dict(dim=2, scaling="base"), dict(dim=8, scaling="parts"),
                dict(dim=8, scaling="parts", original_length=10, low=3.0, high=3.0)):
        with pytest.raises(ValueError):
            F.rotary_frequencies(**bad)


# ---------------------------------------------------------------------------------------- refusals
def tokens(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype)


@pytest.mark.parametrize("case", [
    "rank", "kv shape", "batch", "width", "heads", "width 12", "width 136", "types", "double",
    "scale", "nan scale", "band", "lengths", "lengths type", "mask", "mask type", "no tensor", "host"])
def test_cross_attention_refuses(case):
    q, k = tokens(2, 4, 4, 16), tokens(2, 5, 2, 16)
    v, more, error = k, {}, RuntimeError
    if case == "rank":
        q = q[0]
    elif case == "kv shape":
        v = tokens(2, 6, 2, 16)
    elif case == "batch":
        k = v = tokens(3, 5, 2, 16)
    elif case == "width":
        k = v = tokens(2, 5, 2, 24)
    elif case == "heads":
        k = v = tokens(2, 5, 3, 16)
    elif case in ("width 12", "width 136"):
        d = int(case.split()[1])
        q, k = tokens(2, 4, 4, d), tokens(2, 5, 2, d)
        v = k
    elif case == "types":
        v = k.half()
    elif case == "double":
        q, k = q.double(), k.double()
        v, error = k, TypeError
    elif case == "host":  # everything else is right: there is no host path
        pass
    elif case == "no tensor":
        q, error = [[0.0]], TypeError
    else:
        error = ValueError if case in ("scale", "nan scale", "band") else RuntimeError
        more = {"scale": dict(scale=0.0), "nan scale": dict(scale=math.nan), "band": dict(max_disparity=0),
                "lengths": dict(key_lengths=torch.zeros(3, dtype=torch.int32)),
                "lengths type": dict(key_lengths=torch.zeros(2)),
                "mask": dict(key_mask=torch.zeros(2, 4, dtype=torch.bool)),
                "mask type": dict(key_mask=torch.zeros(2, 5, dtype=torch.uint8))}[case]
    word = {"host": "CPU fallback", "lengths": "key_lengths", "lengths type": "key_lengths", "mask": "key_mask",
            "mask type": "key_mask", "band": "max_disparity"}.get(case, "cross_attention")
    with pytest.raises(error, match=word):
        F.cross_attention(q, k, v, **more)


@pytest.mark.parametrize("case", ["rank", "double", "positions", "float positions", "frequencies",
                                  "too many", "layout", "host"])
def test_rotary_refuses(case):
    x, p, f, layout, error = tokens(2, 3, 1, 8), torch.arange(3), F.rotary_frequencies(8), "half", RuntimeError
    if case == "rank":
        x = x[0]
    elif case == "double":
        x, error = x.double(), TypeError
    elif case == "positions":
        p = torch.arange(4)
    elif case == "float positions":
        p = p.float()
    elif case == "frequencies":
        f = f.float()
    elif case == "too many":
        f = F.rotary_frequencies(10)
    elif case == "layout":
        layout, error = "both", ValueError
    with pytest.raises(error):
        F.rotary(x, p, f, layout=layout)


@pytest.mark.parametrize("case", ["weight", "width", "double", "weight type", "residual type",
                                  "residual shape", "eps", "group", "host", "wide"])
def test_norm_refuses(case):
    x, w, r, eps, error = tokens(2, 8), tokens(8), None, 1e-6, RuntimeError
    if case == "weight":
        w = tokens(7)
    elif case == "width":
        x, w = tokens(2, 0), tokens(0)
    elif case == "wide":
        x, w = tokens(1, 65537), tokens(65537)
    elif case == "double":
        x, error = x.double(), TypeError
    elif case == "weight type":
        w, error = w.half(), TypeError
    elif case == "residual type":
        r, error = tokens(2, 8).half(), TypeError
    elif case == "residual shape":
        r = tokens(3, 8)
    elif case == "eps":
        eps, error = -1.0, ValueError
    elif case == "group":
        with pytest.raises(ValueError):
            F.rms_norm_e4m3(x, w, group=64)
        return
    for f in (F.rms_norm, F.rms_norm_e4m3):
        with pytest.raises(error):
            f(x, w, r, eps)


def _abi(fn, *args):
    lib = _lib.load()
    return getattr(lib, fn)(*args), lib.sm_last_error().decode()


def test_abi_refuses():
    """The C entries return an error before any launch (the pointers are never read)."""
    P = 1 << 20  # a pointer that is 16-byte aligned
    ok = dict(dtype=_lib.SM_BF16, B=1, Lq=4, Lk=8, H=4, KV=2, D=16, scale=0.25, band=0, out=P, q=P, st=None, kst=None,
              ws=None, nws=0)

    def fwd(**kw):
        a = {**ok, **kw}
        return _abi("sm_cross_attention", a["q"], P, P, a["out"], None, a["dtype"], a["B"], a["Lq"], a["Lk"],
                    a["H"], a["KV"], a["D"], a["st"], a["kst"], None, a["scale"], a["band"], None, None, a["ws"],
                    a["nws"], None)

    I3 = ctypes.c_int64 * 3
    for kw, status, word in [
            (dict(dtype=_lib.SM_F64), _lib.SM_EDTYPE, "float32"), (dict(dtype=77), _lib.SM_EDTYPE, "float32"),
            (dict(B=-1), _lib.SM_EINVAL, "negative"), (dict(H=3), _lib.SM_EINVAL, "multiple"),
            (dict(D=12), _lib.SM_EINVAL, "width"), (dict(D=256), _lib.SM_EINVAL, "width"),
            (dict(D=0), _lib.SM_EINVAL, "width"), (dict(KV=0), _lib.SM_EINVAL, "multiple"),
            (dict(scale=0.0), _lib.SM_EINVAL, "scale"), (dict(scale=math.nan), _lib.SM_EINVAL, "scale"),
            (dict(scale=math.inf), _lib.SM_EINVAL, "scale"), (dict(band=-1), _lib.SM_EINVAL, "band"),
            (dict(Lk=1 << 31), _lib.SM_EINVAL, "2^30"), (dict(Lq=1 << 30), _lib.SM_EINVAL, "2^30"),
            (dict(out=None), _lib.SM_EINVAL, "output"), (dict(out=P + 8), _lib.SM_EINVAL, "output"),
            (dict(q=P + 2), _lib.SM_EINVAL, "aligned"), (dict(q=None), _lib.SM_EINVAL, "null"),
            (dict(st=I3(256, 64, 12)), _lib.SM_EINVAL, "strides"), (dict(st=I3(-64, 64, 16)), _lib.SM_EINVAL, "negative"),
            (dict(kst=I3(0, 1 << 23, 16)), _lib.SM_EINVAL, "far apart"),
            (dict(nws=-1), _lib.SM_EINVAL, "workspace"),
            (dict(Lq=1, Lk=8192), _lib.SM_EINVAL, "workspace")]:
        rc, msg = fwd(**kw)
        assert rc == status and word in msg, (kw, rc, msg)
    assert fwd(B=0)[0] == _lib.SM_OK and fwd(Lq=0)[0] == _lib.SM_OK
    assert _lib.load().sm_cross_attention_workspace_bytes(1, 1, 8192, 4, 2, 16) > 0
    assert _lib.load().sm_cross_attention_workspace_bytes(1, 0, 8192, 4, 2, 16) == 0

    def bwd(ws, nws, dout=P, dk=P):
        return _abi("sm_cross_attention_backward", P, P, P, P, P, dout, P, dk, P, _lib.SM_F16, 1, 4, 8, 4, 2,
                    16, None, None, None, None, 0.25, 0, None, None, ws, nws, None)

    n = _lib.load().sm_cross_attention_backward_workspace_bytes(1, 4, 4, 2)
    rc, msg = fwd(B=1 << 29, Lq=1 << 29, H=1 << 19, KV=1 << 19)
    assert rc == _lib.SM_EINVAL and "too large" in msg
    for args, word in [((None, 0), "workspace"), ((P, n - 1), "workspace"), ((P + 4, n), "aligned"),
                       ((P, n, None), "null"), ((P, n, P + 2), "aligned"), ((P, n, P, P + 8), "aligned")]:
        rc, msg = bwd(*args)
        assert rc == _lib.SM_EINVAL and word in msg, (args, rc, msg)

    def rot(dtype=_lib.SM_F16, R=8, flags=0, x=P, D=8, ps=0):
        return _abi("sm_rotary", x, P, P, P, dtype, 1, 2, 1, D, R, None, ps, flags, 1.0, None)

    for kw, status in [(dict(dtype=_lib.SM_F64), _lib.SM_EDTYPE), (dict(R=3), _lib.SM_EINVAL),
                       (dict(R=10), _lib.SM_EINVAL), (dict(R=0), _lib.SM_EINVAL), (dict(flags=8), _lib.SM_EINVAL),
                       (dict(x=None), _lib.SM_EINVAL), (dict(ps=-1), _lib.SM_EINVAL)]:
        assert rot(**kw)[0] == status, kw

    def norm8(dtype=_lib.SM_F16, rt=_lib.SM_F16, wt=_lib.SM_F16, rows=2, C=8, group=0, eps=1e-6, scales=P):
        return _abi("sm_rms_norm_e4m3", P, P, P, P, scales, P, dtype, rt, wt, rows, C, C, C, group, eps, None)

    for kw, status in [(dict(dtype=_lib.SM_F64), _lib.SM_EDTYPE), (dict(rt=_lib.SM_BF16), _lib.SM_EDTYPE),
                       (dict(wt=_lib.SM_BF16), _lib.SM_EDTYPE), (dict(rows=-1), _lib.SM_EINVAL),
                       (dict(C=0), _lib.SM_EINVAL), (dict(C=65537), _lib.SM_EINVAL), (dict(group=64), _lib.SM_EINVAL),
                       (dict(eps=-1.0), _lib.SM_EINVAL), (dict(eps=math.nan), _lib.SM_EINVAL),
                       (dict(scales=None), _lib.SM_EINVAL)]:
        assert norm8(**kw)[0] == status, kw
    rc, msg = _abi("sm_rms_norm_backward", P, P, P, None, P, None, P, _lib.SM_F16, _lib.SM_F16, _lib.SM_F32, 2, 8,
                   8, 8, 8, 1e-6, None, 0, None)
    assert rc == _lib.SM_EINVAL and "workspace" in msg
    rc, msg = _abi("sm_rms_norm_backward", P, P, P, None, P, P, P, _lib.SM_F16, _lib.SM_F16, _lib.SM_F32, 2, 8,
                   8, 8, 8, 1e-6, P, 1 << 20, None)
    assert rc == _lib.SM_EINVAL and "gradient" in msg


# -------------------------------------------------------------------------------- cross attention
# batch, query tokens, key tokens, query heads, key heads, head width, band, mask
ATTENTION = [
    (1, 1, 1, 1, 1, 8, None, None),
    (2, 1, 1, 2, 1, 16, None, "lengths"),
    (1, 3, 31, 1, 1, 32, None, None),
    (2, 33, 32, 2, 2, 40, None, None),
    (1, 32, 33, 4, 2, 64, None, "mask"),
    (2, 64, 63, 2, 1, 64, None, "lengths"),
    (1, 65, 65, 1, 1, 128, None, "both"),
    (2, 127, 129, 3, 3, 96, None, None),
    (1, 129, 127, 6, 2, 128, None, "lengths"),
    (3, 100, 300, 4, 1, 24, None, "both"),
    (2, 257, 70, 5, 1, 72, None, None),
    (2, 128, 128, 1, 1, 32, 24, None),
    (1, 200, 150, 2, 1, 16, 1, None),
    (1, 300, 130, 3, 1, 64, 40, None),        # the last rows' bands lie past the keys
    (2, 150, 260, 2, 2, 128, 192, "both"),
    (2, 90, 97, 4, 2, 56, 64, "lengths"),
    (1, 5, 1500, 6, 1, 64, None, "mask"),      # few rows: the waves split the keys
    (2, 1, 3000, 8, 2, 128, None, "lengths"),  # and the workgroups too
    (1, 1, 2049, 1, 1, 40, None, None),
    (3, 2, 700, 4, 4, 32, None, "both"),
    (1, 40, 2500, 1, 1, 64, None, "mask"),     # ordinary rows, split keys
    (1, 20, 30, 2, 1, 32, 7, "both"),          # few rows in a band
    (2, 40, 1100, 4, 2, 64, None, "both"),     # several tiles of 32 rows, split keys
    (1, 700, 900, 2, 2, 32, 300, None),        # the same in a band: some shares are empty
    (35, 130, 800, 1, 1, 64, None, "both"),    # 128-row tiles, split keys
    # launches of 65 to 256 workgroups of 128 rows or keys: eight waves each
    (20, 130, 140, 4, 4, 64, None, "both"),
    (20, 130, 300, 4, 2, 32, 48, "lengths"),
    (17, 200, 150, 4, 4, 128, None, "mask"),
    (30, 50, 140, 9, 3, 40, None, "lengths"),  # three heads share keys: tiles begin inside a token
    # more than 256: four waves each
    (70, 130, 150, 4, 4, 64, None, "both"),
    (70, 140, 150, 4, 4, 32, 24, "lengths"),
    (70, 130, 135, 4, 4, 128, 30, "mask"),
    (100, 50, 140, 6, 2, 40, 20, "both"),
    (90, 129, 65, 3, 3, 16, None, None),
]


def problem(cfg, dtype, seed=0, holes=math.nan):
    b, lq, lk, h, kv, d, band, kind = cfg
    gen = torch.Generator().manual_seed(seed)
    q = normal(gen, b, lq, h, d, dtype=dtype, scale=1.5)
    k = normal(gen, b, lk, kv, d, dtype=dtype, scale=1.5)
    v = normal(gen, b, lk, kv, d, dtype=dtype)
    g = normal(gen, b, lq, h, d, dtype=dtype)
    lengths = mask = None
    if kind in ("lengths", "both"):  # none, all, one, and anything between
        lengths = torch.randint(0, lk + 1, (b,), generator=gen, dtype=torch.int32)
        lengths[0] = max(1, lk - 3)
        if b > 1:
            lengths[-1] = 0
    if kind in ("mask", "both"):
        mask = torch.rand((b, lk), generator=gen) < 0.7
        mask[0, lk // 2] = True
        if b > 2:
            mask[1] = False
    # what nobody may read holds NaN and infinities
    dead = torch.zeros(b, lk, dtype=torch.bool)
    if lengths is not None:
        dead |= torch.arange(lk)[None] >= lengths[:, None]
    if mask is not None:
        dead |= ~mask
    k, v = k.clone(), v.clone()
    k[dead], v[dead] = holes, holes
    if holes != holes and dead.any():
        v[dead.nonzero()[0][0], dead.nonzero()[0][1]] = math.inf
    return q, k, v, g, lengths, mask


def cuda(*ts):
    return [t.cuda() if isinstance(t, torch.Tensor) else t for t in ts]


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=name)
@pytest.mark.parametrize("cfg", ATTENTION, ids=lambda c: "-".join(map(str, c)))
def test_cross_attention(cfg, dtype):
    b, lq, lk, h, kv, d, band, kind = cfg
    q, k, v, g, lengths, mask = problem(cfg, dtype)
    ok = O.allowed(b, lq, lk, band, lengths, mask)
    val, tol = O.attention(q, k, v, d ** -0.5, ok, g)
    Q, K, V, G, LN, M = cuda(q, k, v, g, lengths, mask)
    how = dict(max_disparity=band, key_lengths=LN, key_mask=M)
    out, lse = F.cross_attention(Q, K, V, return_lse=True, **how)
    near(lse, val["lse"], tol["lse"], "lse")
    near(out, val["out"], tol["out"], "out")
    Q, K, V = (x.requires_grad_() for x in (Q, K, V))
    out2 = F.cross_attention(Q, K, V, **how)
    assert torch.equal(out, out2)
    grads = torch.autograd.grad(out2, (Q, K, V), G)
    for n, x in zip(("dq", "dk", "dv"), grads):
        near(x, val[n], tol[n], n)


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=name)
def test_cross_attention_scale_and_lengths_types(dtype):
    cfg = (2, 50, 70, 2, 1, 48, None, "lengths")
    q, k, v, g, lengths, _ = problem(cfg, dtype, seed=3)
    val, tol = O.attention(q, k, v, 0.03, O.allowed(2, 50, 70, None, lengths), g)
    Q, K, V = cuda(q, k, v)
    for t in (torch.int32, torch.int64):
        near(F.cross_attention(Q, K, V, scale=0.03, key_lengths=lengths.cuda().to(t)), val["out"], tol["out"], t)
    # lengths past the keys and below 0 are taken into their range
    wild = torch.tensor([1 << 40, -(1 << 40)]).cuda()
    wild32 = torch.tensor([1 << 30, -5], dtype=torch.int32).cuda()
    val, tol = O.attention(q, torch.nan_to_num(k, 0.0), torch.nan_to_num(v, 0.0, 0.0), 0.03,
                           O.allowed(2, 50, 70, None, torch.tensor([70, 0])))
    for w in (wild, wild32):
        near(F.cross_attention(Q, *cuda(torch.nan_to_num(k, 0.0), torch.nan_to_num(v, 0.0, 0.0)), scale=0.03,
                               key_lengths=w), val["out"], tol["out"], "wild")


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=name)
def test_cross_attention_strides(dtype):
    """Head-major storage, slices of wider rows, rows that are not aligned, broadcast batches and
    gradients that are one value everywhere."""
    gen = torch.Generator().manual_seed(5)
    q = normal(gen, 2, 4, 45, 32, dtype=dtype)            # (B, H, L, D)
    kvp = normal(gen, 2, 50, 2, 2, 40, dtype=dtype)       # keys and values side by side
    scale = 32 ** -0.5
    Q = q.cuda().transpose(1, 2)
    for lo in (0, 3, 8):
        KV = kvp.cuda()[..., lo:lo + 32]
        K, V = KV[:, :, 0], KV[:, :, 1]
        k, v = K.cpu(), V.cpu()
        val, tol = O.attention(q.transpose(1, 2), k, v, scale, O.allowed(2, 45, 50), torch.ones(2, 45, 4, 32))
        Ql, Kl, Vl = (x.detach().requires_grad_() for x in (Q, K, V))
        out = F.cross_attention(Ql, Kl, Vl)
        near(out, val["out"], tol["out"], lo)
        for n, x in zip(("dq", "dk", "dv"), torch.autograd.grad(out.sum(), (Ql, Kl, Vl))):
            near(x, val[n], tol[n], (lo, n))
    one = kvp.cuda()[:1, :, 0, :, :32]
    val, tol = O.attention(q.transpose(1, 2), one.cpu().expand(2, -1, -1, -1), one.cpu().expand(2, -1, -1, -1),
                           scale, O.allowed(2, 45, 50), torch.ones(2, 45, 4, 32))
    leaf = one.detach().clone().requires_grad_()
    out = F.cross_attention(Q, leaf.expand(2, -1, -1, -1), leaf.expand(2, -1, -1, -1))
    near(out, val["out"], tol["out"], "broadcast")
    grad, = torch.autograd.grad(out.sum(), leaf)
    want = val["dk"].sum(0, keepdim=True) + val["dv"].sum(0, keepdim=True)
    bound = tol["dk"].sum(0, keepdim=True) + tol["dv"].sum(0, keepdim=True)
    # autograd adds four 16-bit tensors: three more roundings of partial sums
    more = 3 * O.unit(dtype) * (val["dk"].abs() + val["dv"].abs()).sum(0, keepdim=True)
    near(grad, want, bound + more, "broadcast grad")


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=name)
def test_cross_attention_empty(dtype):
    e = lambda *s: torch.zeros(s, dtype=dtype, device="cuda", requires_grad=True)  # noqa: E731
    for b, lq, lk in ((0, 3, 4), (2, 0, 4), (2, 3, 0)):
        q, k, v = e(b, lq, 2, 16), e(b, lk, 1, 16), e(b, lk, 1, 16)
        out, lse = F.cross_attention(q, k, v, return_lse=True)
        assert out.shape == (b, lq, 2, 16) and not out.any() and bool((lse == -math.inf).all())
        for x, y in zip((q, k, v), torch.autograd.grad(out.sum(), (q, k, v))):
            assert x.shape == y.shape and not y.any()


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=name)
def test_cross_attention_large_scores(dtype):
    """Scores far apart, rising from key to key (the running maximum moves at every tile) and falling:
    the output is one value row.  Neighbouring keys differ by 128 in the exponent, so every other
    weight is 0 and the row's sum is the one weight w = 2^r, |r| <= 2^-24 |m c| the rounding of the
    product m c that the exponent subtracts.  The output is fl(fl(round(w) v) fl(1 / w)): three fp32
    roundings, and in 16 bits the weight's rounding as an operand and the output's."""
    lk = 200
    k = torch.zeros(1, lk, 1, 16, dtype=dtype)
    k[0, :, 0, 0] = torch.arange(lk) * 2.0
    v = normal(torch.Generator().manual_seed(9), 1, lk, 1, 16, dtype=dtype)
    q = torch.zeros(1, 80, 1, 16, dtype=dtype)
    q[0, :, 0, 0] = torch.where(torch.arange(80) % 2 == 0, 64.0, -64.0)
    out = F.cross_attention(*cuda(q, k, v), scale=1.0).cpu()
    u = 0.0 if dtype == torch.float32 else O.unit(dtype)
    for got, row in ((out[0, 0::2, 0], v[0, -1]), (out[0, 1::2, 0], v[0, 0])):
        want = row.double().expand(40, -1)
        near(got, want, (2.001 * u + 4 * O.F32) * want.abs() + O.tiny(dtype), "row")


@gpu
def test_cross_attention_small_fp16_gradients():
    """Gradients of 2^-12 and below, where p (g.v - delta) is under fp16's range."""
    cfg = (1, 96, 400, 2, 1, 64, None, None)
    q, k, v, g, _, _ = problem(cfg, torch.float16, seed=4)
    q, g = q * 0.1, (g.float() * 2.0 ** -12).half()
    val, tol = O.attention(q, k, v, 0.125, O.allowed(1, 96, 400), g)
    Q, K, V, G = cuda(q, k, v, g)
    Q, K, V = (x.requires_grad_() for x in (Q, K, V))
    for n, x in zip(("dq", "dk", "dv"), torch.autograd.grad(F.cross_attention(Q, K, V), (Q, K, V), G)):
        near(x, val[n], tol[n], n)


@gpu
@pytest.mark.parametrize("lq", [1, 40])
def test_cross_attention_far_offsets(lq):
    """Keys 2^23 - 2^16 values apart: the last one lies past 2^32 bytes and 2^31 values."""
    apart, lk, d = (1 << 23) - (1 << 16), 300, 64
    store = torch.empty(lk * apart, dtype=torch.bfloat16, device="cuda")
    gen = torch.Generator().manual_seed(6)
    q, k, v = (normal(gen, 1, n, 1, d, dtype=torch.bfloat16) for n in (lq, lk, lk))
    K = torch.as_strided(store, (1, lk, 1, d), (lk * apart, apart, d, 1))
    V = torch.as_strided(store, (1, lk, 1, d), (lk * apart, apart, d, 1), 4096)
    K.copy_(k)
    V.copy_(v)
    g = normal(gen, 1, lq, 1, d, dtype=torch.bfloat16)
    val, tol = O.attention(q, k, v, d ** -0.5, O.allowed(1, lq, lk), g)
    Q = q.cuda().requires_grad_()
    K.requires_grad_()
    out = F.cross_attention(Q, K, V)
    near(out, val["out"], tol["out"], "out")
    dq, dk = torch.autograd.grad(out, (Q, K), g.cuda())
    near(dq, val["dq"], tol["dq"], "dq")
    near(dk, val["dk"], tol["dk"], "dk")


@gpu
@pytest.mark.parametrize("cfg", [(2, 130, 200, 4, 2, 64, 48, "both"), (2, 1, 1500, 4, 1, 128, None, "lengths")],
                         ids=["rows", "token"])
def test_cross_attention_graph_and_streams(cfg):
    """Captured once with its gradients, replayed with new inputs between eager calls; and called on
    another stream.  The same bits each time."""
    band = cfg[6]
    sets = [cuda(*problem(cfg, torch.bfloat16, seed=s)) for s in range(3)]
    static = [None if t is None else t.clone() for t in sets[0]]
    leaves = [t.requires_grad_() for t in static[:3]]

    def step():
        out = F.cross_attention(*leaves, max_disparity=band, key_lengths=static[4], key_mask=static[5])
        return (out.detach(), *torch.autograd.grad(out, leaves, static[3]))

    def eager(s):
        ls = [t.detach().clone().requires_grad_() for t in s[:3]]
        out = F.cross_attention(*ls, max_disparity=band, key_lengths=s[4], key_mask=s[5])
        return [out.detach(), *torch.autograd.grad(out, ls, s[3])]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for s in (0, 1, 2, 1):
        with torch.no_grad():
            for x, y in zip(static, sets[s]):
                if x is not None:
                    x.copy_(y)
        graph.replay()
        want = eager(sets[s])
        torch.cuda.synchronize()
        for x, y in zip(held, want):
            assert torch.equal(x, y)
    with torch.cuda.stream(side):
        other = eager(sets[2])
    side.synchronize()
    for x, y in zip(other, eager(sets[2])):
        assert torch.equal(x, y)


# ------------------------------------------------------------------------------------------ rotary
ROTARY = [  # batch, length, heads, width, turned values
    (1, 1, 1, 2, 2), (2, 5, 3, 8, 4), (2, 3, 2, 10, 6), (1, 7, 1, 32, 32), (3, 1, 32, 128, 128),
    (2, 33, 4, 64, 16), (1, 65, 2, 80, 80), (2, 40, 5, 96, 48), (1, 3000, 16, 128, 64)]


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=name)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("cfg", ROTARY, ids=lambda c: "-".join(map(str, c)))
def test_rotary(cfg, layout, dtype):
    b, l, h, d, r = cfg
    gen = torch.Generator().manual_seed(11)
    x, g = normal(gen, b, l, h, d, dtype=dtype), normal(gen, b, l, h, d, dtype=dtype)
    f = F.rotary_frequencies(r) if r > 2 else torch.ones(1, dtype=torch.float64)
    X = x.cuda().requires_grad_()
    for positions in (torch.arange(l), torch.randint(-(1 << 31), 1 << 31, (b, l), generator=gen),
                      torch.randint(0, 1 << 20, (b, l), generator=gen, dtype=torch.int32)):
        y = F.rotary(X, positions.cuda(), f.cuda(), layout=layout, amplitude=1.25)
        want, tol = O.rotary(x, positions, f, layout, 1.25)
        near(y, want, tol, "y")
        dx, = torch.autograd.grad(y, X, g.cuda())
        want, tol = O.rotary(g, positions, f, layout, 1.25, inverse=True)
        near(dx, want, tol, "dx")


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=name)
def test_rotary_strides_and_empty(dtype):
    gen = torch.Generator().manual_seed(12)
    f = F.rotary_frequencies(16)
    wide = normal(gen, 2, 3, 9, 40, dtype=dtype)  # (B, H, L, D + more)
    p = torch.arange(18).view(9, 2)[:, 0] * 7      # every second value
    for lo in (0, 1, 8):
        x = wide[..., lo:lo + 24].transpose(1, 2)
        X = wide.cuda()[..., lo:lo + 24].transpose(1, 2)
        near(F.rotary(X, torch.arange(18).cuda().view(9, 2)[:, 0] * 7, f.cuda()), *O.rotary(x, p, f, "half"), lo)
    x = wide[:, :, :, :24].permute(0, 2, 3, 1)      # the values are not neighbours
    X = wide.cuda()[:, :, :, :24].permute(0, 2, 3, 1)
    f1 = torch.ones(1, dtype=torch.float64)
    near(F.rotary(X, torch.arange(9).cuda(), f1.cuda()), *O.rotary(x, torch.arange(9), f1, "half"), "permuted")
    for shape in ((0, 4, 1, 16), (2, 0, 1, 16), (2, 4, 0, 16)):
        e = torch.zeros(shape, dtype=dtype, device="cuda", requires_grad=True)
        y = F.rotary(e, torch.arange(shape[1]).cuda(), f.cuda())
        assert y.shape == shape and torch.autograd.grad(y.sum(), e)[0].shape == shape


# -------------------------------------------------------------------------------------------- norm
NORM = [(1, 1), (3, 7), (5, 8), (33, 32), (70, 64), (9, 100), (40, 128), (11, 250), (130, 256), (3, 512),
        (2, 513), (5, 1000), (4, 2048), (3, 2056), (2, 4099), (3, 5000), (2, 8192), (1, 8200), (2, 20000),
        (1, 65536), (2100, 64), (40, 1000)]


def norm_inputs(rows, c, dtype, residual, weight, seed=21):
    gen = torch.Generator().manual_seed(seed)
    x = normal(gen, rows, c, dtype=dtype)
    w = (1 + 0.3 * torch.randn(c, generator=gen)).to(weight)
    r = None if residual is None else normal(gen, rows, c, dtype=residual, scale=2.0)
    g = normal(gen, rows, c, dtype=dtype)
    z = None if residual is None else normal(gen, rows, c, dtype=residual)
    return x, w, r, g, z


def kinds(dtype):
    wide = torch.float32
    return [(None, dtype), (dtype, wide), (wide, dtype)] if dtype != wide else [(None, wide), (wide, wide)]


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=name)
@pytest.mark.parametrize("rows,c", NORM)
def test_rms_norm(rows, c, dtype):
    for residual, weight in kinds(dtype):
        x, w, r, g, z = norm_inputs(rows, c, dtype, residual, weight)
        val, tol = O.rms_norm(x, w, r, 1e-5, g, z)
        X, W, R, G, Z = cuda(x, w, r, g, z)
        leaves = [t.requires_grad_() for t in (X, W, R) if t is not None]
        if r is None:
            y = F.rms_norm(X, W, eps=1e-5)
            grads = torch.autograd.grad(y, leaves, G)
        else:
            y, s = F.rms_norm(X, W, R, eps=1e-5)
            near(s, val["summed"], tol["summed"], "summed")
            grads = torch.autograd.grad((y, s), leaves, (G, Z))
            near(grads[2], val["dx"], tol["dx"] + O.unit(residual) * val["dx"].abs() + O.tiny(residual), "dresidual")
        near(y, val["y"], tol["y"], "y")
        near(grads[0], val["dx"], tol["dx"] + O.unit(dtype) * val["dx"].abs() + O.tiny(dtype), "dx")
        near(grads[1], val["dweight"], tol["dweight"], "dweight")


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=name)
@pytest.mark.parametrize("group", [None, 128])
@pytest.mark.parametrize("rows,c", NORM)
def test_rms_norm_e4m3(rows, c, group, dtype):
    """q * scale against y: scale within the norm's bound, q off by half a step of e4m3 (2^-4, or 2^-10
    below 2^-6) of y / scale, which itself is off by the bounds of y and of the scale."""
    for residual, weight in kinds(dtype):
        x, w, r, _, _ = norm_inputs(rows, c, dtype, residual, weight)
        val, _ = O.rms_norm(x, w, r, 1e-5)
        got = F.rms_norm_e4m3(*cuda(x, w, r), eps=1e-5, group=group)
        assert len(got) == (2 if r is None else 3)
        q, scale = got[0], got[1]
        assert q.dtype == torch.float8_e4m3fn and scale.dtype == torch.float32
        if r is not None:
            assert torch.equal(got[2].cpu().double(), val["summed"])
        parts = val["y"].split(group or c, -1)
        top = torch.stack([p.abs().amax(-1) for p in parts], -1)
        want = torch.where(top == 0, 448.0, top) / 448
        rel = (c / 2 + 14) * O.F32
        near(scale.view(want.shape), want, rel * want, "scale")
        z = torch.cat([p / want[:, i:i + 1] for i, p in enumerate(parts)], -1)
        near(q.float(), z, (2.0 ** -4 + 2 * rel) * z.abs() + 2.0 ** -10, "q")
        # the largest value of a group is held by the largest code
        assert bool((torch.stack([p.abs().amax(-1) for p in q.cpu().float().split(group or c, -1)], -1) >= 416).all())


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=name)
@pytest.mark.parametrize("group", [None, 128])
@pytest.mark.parametrize("rows,c", [(6000, 1000), (40000, 64), (700, 5000), (60, 20000)])
def test_rms_norm_e4m3_codes(rows, c, group, dtype):
    """s w 448 / max |s w| in 64 bits, rounded to 32 and then to 8: none of a million codes differs (the
    kernel's 64-bit value is within 4 units of 2^-53, which decides a rounding to 32 bits once in 2^27)."""
    for kind in kinds(dtype):
        x, w, r, _, _ = norm_inputs(rows, c, dtype, *kind, seed=c)
        s = x if r is None else (x.double() + r.double()).to(r.dtype)
        sw = s.double() * w.double()
        parts = sw.split(group or c, -1)
        want = torch.cat([(p * (448 / p.abs().amax(-1, keepdim=True))).float().to(torch.float8_e4m3fn)
                          for p in parts], -1)
        q = F.rms_norm_e4m3(*cuda(x, w, r), group=group)[0].cpu()
        differ = int((q.view(torch.uint8) != want.view(torch.uint8)).sum())
        assert differ == 0, (kind, differ)


@gpu
def test_rms_norm_special_rows():
    """Rows of zeros, of one value, with NaN or infinity: they stay in their rows."""
    x = torch.ones(6, 300, device="cuda")
    x[1] = 0
    x[2, 5] = math.nan
    x[3, 7] = math.inf
    x[4] = 1e-30
    w = torch.ones(300, device="cuda")
    y = F.rms_norm(x, w, eps=0.0)
    # 1 / sqrt(1): two roundings; the row of 1e-30 underflows in its squares, as in the plain form
    assert bool(((y[0] - 1).abs() <= 4 * O.F32).all()) and torch.equal(y[5], y[0])
    assert bool(y[2].isnan().all()) and bool(y[3, 7].isnan())
    q, s = F.rms_norm_e4m3(x, w)
    assert not q[1].float().any() and s[1] == 1.0
    assert bool(s[2].isnan()) and bool(q[2].float().isnan().all())
    assert bool((q[0].float() == 448).all()) and torch.equal(q[5].float(), q[0].float())


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=name)
def test_rms_norm_shapes_and_strides(dtype):
    gen = torch.Generator().manual_seed(31)
    wide = normal(gen, 3, 5, 2, 50, dtype=dtype)
    w = normal(gen, 40, dtype=torch.float32)
    for lo in (0, 3, 8):
        x = wide[..., lo:lo + 40]
        X = wide.cuda()[..., lo:lo + 40]
        val, tol = O.rms_norm(x, w, x, 1e-6)
        y, s = F.rms_norm(X, w.cuda(), X)
        assert y.shape == x.shape
        near(y, val["y"], tol["y"], lo)
        near(s, val["summed"], tol["summed"], lo)
    one = normal(gen, 1, 40, dtype=dtype)
    X = one.cuda().requires_grad_()
    y = F.rms_norm(X.expand(9, 40), w.cuda())
    val, tol = O.rms_norm(one.expand(9, 40), w, None, 1e-6, torch.ones(9, 40))
    dx, = torch.autograd.grad(y.sum(), X)
    # autograd adds nine equal 16-bit rows: eight roundings of partial sums
    bound = (tol["dx"] + 9 * O.unit(dtype) * val["dx"].abs()).sum(0, keepdim=True) + 9 * O.tiny(dtype)
    near(dx, val["dx"].sum(0, keepdim=True), bound, "broadcast")
    for shape in ((0, 40), (2, 0, 40)):
        e = torch.zeros(shape, dtype=dtype, device="cuda", requires_grad=True)
        W = w.cuda().requires_grad_()
        y = F.rms_norm(e, W)
        assert y.shape == shape
        de, dw = torch.autograd.grad(y.sum(), (e, W))
        assert de.shape == shape and not dw.any()
        q, s = F.rms_norm_e4m3(e.detach(), w.cuda(), group=128)
        assert q.shape == shape and s.shape == (*shape[:-1], 1)


@gpu
def test_rms_norm_only_stream_used():
    x, r = torch.randn(4, 16, device="cuda", requires_grad=True), torch.randn(4, 16, device="cuda", requires_grad=True)
    w = torch.ones(16, device="cuda", requires_grad=True)
    _, s = F.rms_norm(x, w, r)
    dx, dr = torch.autograd.grad(s.sum(), (x, r))
    assert torch.equal(dx, torch.ones_like(x)) and torch.equal(dr, dx)
    y, _ = F.rms_norm(x, w, r)
    val, tol = O.rms_norm(x, w, r, 1e-6, torch.ones(4, 16))
    dx, = torch.autograd.grad(y.sum(), x)
    near(dx, val["dx"], tol["dx"] + O.F32 * val["dx"].abs(), "dx")


@gpu
def test_rms_norm_e4m3_is_forward_only():
    x = torch.ones(2, 8, device="cuda", requires_grad=True)
    with pytest.raises(NotImplementedError):
        F.rms_norm_e4m3(x, torch.ones(8, device="cuda"))
    with torch.no_grad():
        F.rms_norm_e4m3(x, torch.ones(8, device="cuda"))


# ------------------------------------------------------------------------------ a layer, and tracing
def layer(norm, rot, attend, left, right, res_l, res_r, w, wq, wk, wv, wo, f):
    """One matching layer on feature rows: norm, projections, rotary, banded cross attention, and the
    next layer's norm.  (rows, tokens, C)."""
    x, stream = norm(left, w, res_l)
    y, _ = norm(right, w, res_r)
    heads = lambda t, m: (t @ m).unflatten(-1, (2, 16))  # noqa: E731
    i, j = torch.arange(x.shape[1], device=x.device), torch.arange(y.shape[1], device=x.device)
    o = attend(rot(heads(x, wq), i, f), rot(heads(y, wk), j, f), heads(y, wv))
    return norm(o.flatten(2) @ wo, w, stream)


def layer_inputs(dtype, device):
    gen = torch.Generator().manual_seed(41)
    n = lambda *s, scale=1.0: normal(gen, *s, scale=scale).to(device, dtype).requires_grad_()  # noqa: E731
    return [n(3, 40, 32), n(3, 47, 32), n(3, 40, 32), n(3, 47, 32), n(32),
            *(n(32, 32, scale=0.2) for _ in range(4))]


def _plain_layer(ins):
    def norm(x, w, r):
        s = x + r
        return s / (s.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w, s

    def rot(x, p, f):
        z = torch.polar(torch.ones((), dtype=torch.float64), p.double()[:, None] * f)[:, None]
        t = torch.complex(x[..., :8], x[..., 8:]) * z
        return torch.cat((t.real, t.imag), -1)

    def attend(q, k, v):
        q, k, v = (t.transpose(1, 2) for t in (q, k, v))
        s = q @ k.transpose(2, 3) * 0.25
        d = torch.arange(q.shape[2])[:, None] - torch.arange(k.shape[2])
        p = s.masked_fill((d < 0) | (d >= 12), -math.inf).softmax(-1)
        return (p @ v).transpose(1, 2)

    return layer(norm, rot, attend, *ins, F.rotary_frequencies(16))


@gpu
def test_matching_layer():
    """The operators together, with all gradients, in fp32 against 64 bits: 1e-5 of each tensor's norm
    (some thirty chained fp32 sums of up to 47 terms: 30 * 47 * 2^-24 = 8.4e-5 at the very worst, all
    one way; 1e-5 is what independent signs leave with a factor of four to spare)."""
    ins64 = layer_inputs(torch.float64, "cpu")
    y, s = _plain_layer(ins64)
    want = [y, s, *torch.autograd.grad((y.sin().sum() + s.cos().sum()), ins64)]
    ins = layer_inputs(torch.float32, "cuda")
    got = layer(lambda x, w, r: F.rms_norm(x, w, r), F.rotary,
                lambda q, k, v: F.cross_attention(q, k, v, max_disparity=12), *ins,
                F.rotary_frequencies(16, device="cuda"))
    grads = torch.autograd.grad(got[0].sin().sum() + got[1].cos().sum(), ins)
    for n, (x, z) in enumerate(zip((*got, *grads), want)):
        off = (x.detach().cpu().double() - z.detach()).norm() / z.detach().norm()
        assert off < 1e-5, (n, float(off))


def test_matching_ops_fake():
    from torch._subclasses.fake_tensor import FakeTensorMode

    from realtime_stereo_matcher_amd import library  # noqa: F401
    ops = torch.ops.stereocv
    with FakeTensorMode():
        q, k = torch.empty(2, 5, 4, 16, dtype=torch.half), torch.empty(2, 7, 2, 16, dtype=torch.half)
        out, lse = ops.cross_attention(q, k, k)
        assert out.shape == q.shape and out.dtype == q.dtype and lse.shape == (2, 2, 10) and lse.dtype == torch.float32
        dq, dk, dv = ops.cross_attention_backward(q, k, k, out, lse, out)
        assert dq.shape == q.shape and dk.shape == dv.shape == k.shape
        assert ops.rotary(q, torch.arange(5), torch.empty(8, dtype=torch.float64)).shape == q.shape
        x, w, r = torch.empty(3, 200, dtype=torch.half), torch.empty(200), torch.empty(3, 200)
        assert ops.rms_norm(x, w).dtype == torch.half
        y, s = ops.add_rms_norm(x, w, r)
        assert y.dtype == torch.half and s.dtype == torch.float32
        q8, sc = ops.rms_norm_e4m3(x, w, 1e-6, 128)
        assert q8.dtype == torch.float8_e4m3fn and sc.shape == (3, 2)
        assert ops.add_rms_norm_e4m3(x, w, r)[1].shape == (3, 1)
        dx, dr, dw = ops.rms_norm_backward(r, w, x)
        assert dx.dtype == torch.half and dr.shape == r.shape and dw.shape == w.shape


@gpu
def test_matching_ops_traced():
    """jit.trace holds the operators, and compiled-style calls of torch.ops give the eager gradients."""
    from realtime_stereo_matcher_amd import library  # noqa: F401
    f = F.rotary_frequencies(16, device="cuda")

    class Net(torch.nn.Module):
        def forward(self, x, y, w):
            a, s = F.rms_norm(x, w, x)
            a = F.rotary(a.unflatten(-1, (2, 16)), torch.arange(20, device="cuda"), f)
            b = F.rms_norm(y, w).unflatten(-1, (2, 16))
            return F.cross_attention(a, b, b, max_disparity=9).flatten(2) + s

    gen = torch.Generator().manual_seed(51)
    ins = [normal(gen, 2, 20, 32).cuda(), normal(gen, 2, 23, 32).cuda(), normal(gen, 32).cuda()]
    net = Net()
    with torch.no_grad():
        traced = torch.jit.trace(net, [torch.randn_like(t) for t in ins])
    text = str(traced.inlined_graph)
    for op in ("cross_attention", "rotary", "add_rms_norm", "rms_norm"):
        assert f"stereocv::{op}" in text
    assert torch.equal(traced(*ins), net(*ins))
    ops = torch.ops.stereocv
    q, k, v = (normal(gen, 2, n, 2, 16).cuda().requires_grad_() for n in (9, 11, 11))
    got = torch.autograd.grad(ops.cross_attention(q, k, v, None, None, None, 5)[0].sin().sum(), (q, k, v))
    want = torch.autograd.grad(F.cross_attention(q, k, v, max_disparity=5).sin().sum(), (q, k, v))
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    p = torch.arange(9, device="cuda")
    got, = torch.autograd.grad(ops.rotary(q, p, f[:4], "interleaved").sin().sum(), q)
    want, = torch.autograd.grad(F.rotary(q, p, f[:4], layout="interleaved").sin().sum(), q)
    assert torch.equal(got, want)
    for res in (None, torch.float32, torch.float16):
        x = normal(gen, 4, 40, dtype=torch.float16).cuda().requires_grad_()
        w = normal(gen, 40).cuda().requires_grad_()
        if res is None:
            got = torch.autograd.grad(ops.rms_norm(x, w, 1e-6).sin().sum(), (x, w))
            want = torch.autograd.grad(F.rms_norm(x, w).sin().sum(), (x, w))
        else:
            r = normal(gen, 4, 40, dtype=res).cuda().requires_grad_()
            y, s = ops.add_rms_norm(x, w, r, 1e-6)
            got = torch.autograd.grad(y.sin().sum() + s.cos().sum(), (x, w, r))
            y, s = F.rms_norm(x, w, r)
            want = torch.autograd.grad(y.sin().sum() + s.cos().sum(), (x, w, r))
        assert all(torch.equal(x, y) for x, y in zip(got, want))
