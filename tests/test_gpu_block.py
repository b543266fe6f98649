"""ftb.block_norm, rms_norm, rope and rope_append against their definitions in 64 bits.

Bounds, elementwise, with u the unit roundoff of the output's type (2^-8 bf16, 2^-11 f16, 2^-24
f32): every step is fp32, each output is rounded once. The mean square is a sum of H <= 2^14
squares in fp32, in chunks and a tree: at most 2^-24 * 64 relative, halved by the square root, and
rsqrt, the products and the gate's sigmoid add a few 2^-23: n is good to 2^-18 relative.
  r = x + a n:  u |r| + 2^-18 |a n| + 2^-23 |r|
  h = r s w:    u |h| + (2^-18 |h| + 2^-18 max |a n| s |w|)
  rope:         u |out| + 2^-22 (|a| + |b|)
f16 and bf16 outputs below the normal range: 2^-25 more (f16).
"""
import math

import pytest
import torch

import ftb

pytestmark = pytest.mark.gpu
BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32
U = {BF: 2.0 ** -8, F16: 2.0 ** -11, F32: 2.0 ** -24}


def ref_norm(x, y, post, gate, scale, pre, eps, act):
    x = x.double()
    n, r = torch.zeros_like(x), x
    if y is not None:
        n = y.double()
        if post is not None:
            n = n / (n.square().mean(-1, keepdim=True) + eps).sqrt() * post.double()
        if gate is not None:
            n = n * (gate.double().sigmoid() if act == "sigmoid" else gate.double())
        n = n * scale
        r = x + n
    h = b = None
    if pre is not None:
        s = 1 / (r.square().mean(-1, keepdim=True) + eps).sqrt()
        h = r * s * pre.double()
        b = 2.0 ** -18 * (h.abs() + n.abs() * s * pre.double().abs())
        b = b + 2.0 ** -18 * h.abs()
    return r, 2.0 ** -18 * n.abs() + 2.0 ** -23 * r.abs(), h, b


def near(got, ref, bound):
    tiny = 2.0 ** -25 if got.dtype == F16 else 1e-38
    lim = U[got.dtype] * ref.abs() + bound * 1.01 + tiny
    bad = ((got.double() - ref).abs() / lim).max().item() if ref.numel() else 0
    assert bad <= 1.0, bad


def run_norm(rows, H, dtype, res, gate=None, act=None, post=True, pre=True, wf32=False, seed=0,
             scale=0.5, strided=False):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def rnd(*shape, dtype=dtype, s=1.0, m=0.0):
        return (torch.randn(*shape, generator=g, device="cuda") * s + m).to(dtype)

    w = F32 if wf32 else dtype
    width = H + 24 if strided else H
    x, y = rnd(rows, width, dtype=res, s=3.0)[:, :H], rnd(rows, width)[:, :H]
    post_w = rnd(H, dtype=w, s=0.1, m=1.0) if post else None
    pre_w = rnd(H, dtype=w, s=0.1, m=1.0) if pre else None
    shape = {None: None, "channel": (H,), "token": (rows, 1), "full": (rows, H)}[gate]
    gt = rnd(*shape, dtype=w) if shape else None
    r, h = ftb.block_norm(x, y, post_weight=post_w, gate=gt, scale=scale, pre_weight=pre_w,
                          gate_act=act)
    assert r.dtype == res and (h is None) == (not pre)
    rr, rb, rh, hb = ref_norm(x, y, post_w, gt, scale, pre_w, 1e-6, act)
    near(r, rr, rb)
    if pre:
        assert h.dtype == dtype
        near(h, rh, hb)


@pytest.mark.parametrize("dtype,res", [(BF, BF), (BF, F32), (F16, F16), (F16, F32)])
@pytest.mark.parametrize("H", [1, 7, 8, 64, 100, 255, 256, 1000, 2045, 2048, 4096, 4097, 5000,
                               8192, 16383, 16384])
def test_block_norm_widths(H, dtype, res):
    run_norm(5, H, dtype, res, seed=H)


@pytest.mark.parametrize("rows", [1, 2, 7, 8, 9, 64, 1021, 5000])
def test_block_norm_rows(rows):
    run_norm(rows, 192, BF, BF, gate="token")
    run_norm(rows, 2048, BF, F32, gate="channel")


@pytest.mark.parametrize("gate", [None, "channel", "token", "full"])
@pytest.mark.parametrize("act", [None, "sigmoid"])
@pytest.mark.parametrize("wf32", [False, True])
@pytest.mark.parametrize("H", [1024, 333])
def test_block_norm_gates(gate, act, wf32, H):
    run_norm(33, H, BF, F32, gate, act, wf32=wf32)
    run_norm(33, H, F16, F16, gate, act, post=False, wf32=wf32)
    run_norm(33, H, BF, BF, gate, act, pre=False, wf32=wf32)


def test_block_norm_strided_rows():
    run_norm(40, 512, BF, BF, gate="full", strided=True)
    run_norm(40, 511, F16, F32, strided=True)


def test_block_norm_in_place():
    g = torch.Generator(device="cuda").manual_seed(1)
    for H in (4096, 777):
        x = torch.randn(50, H, generator=g, device="cuda").to(BF)
        y = torch.randn(50, H, generator=g, device="cuda").to(BF)
        w = torch.ones(H, dtype=BF, device="cuda")
        r, h = ftb.block_norm(x, y, post_weight=w, pre_weight=w)
        r2, h2 = ftb.block_norm(x, y, post_weight=w, pre_weight=w, residual_out=x, out=y)
        assert r2 is x and h2 is y and torch.equal(x, r) and torch.equal(y, h)


def test_rms_norm():
    g = torch.Generator(device="cuda").manual_seed(2)
    for shape in ((3, 5, 640), (1, 4096), (77,)):
        x = torch.randn(*shape, generator=g, device="cuda").to(BF)
        w = torch.randn(shape[-1], generator=g, device="cuda").to(BF)
        h = ftb.rms_norm(x, w)
        _, _, ref, b = ref_norm(x, None, None, None, 1, w, 1e-6, None)
        near(h, ref, b)


def test_norm_extremes():
    """Zero rows stay zero (eps), infinities and NaN stay in their rows, f16 squares past f16."""
    x = torch.zeros(4, 256, dtype=F16, device="cuda")
    x[1] = 60000.0
    x[2, 3] = math.inf
    x[3, 7] = math.nan
    w = torch.ones(256, dtype=F16, device="cuda")
    h = ftb.rms_norm(x, w)
    assert (h[0] == 0).all() and (h[1] == 1).all()
    assert torch.isnan(h[2, 3]) and (h[2, :3] == 0).all() and torch.isnan(h[3]).all()


def test_norm_refusals():
    x = torch.zeros(4, 64, dtype=BF, device="cuda")
    w = torch.ones(64, dtype=BF, device="cuda")

    def refuse(*a, **kw):
        with pytest.raises((ValueError, ftb._lib.FtbError)):
            ftb.block_norm(*a, **kw)

    refuse(x, x.float())
    refuse(x.half(), x)
    refuse(x, x[:2])
    refuse(x, x, pre_weight=w[:32])
    refuse(x, x, pre_weight=w.double())
    refuse(x, x, pre_weight=w, post_weight=w.float())
    refuse(x, x, gate=w[:3])
    refuse(x, x, gate=w, gate_act="tanh")
    refuse(x, x, pre_weight=w, out=x.float())
    refuse(x.cpu(), x.cpu())
    refuse(x, x.t().contiguous().t())
    wide = torch.zeros(2, 16385, dtype=BF, device="cuda")
    refuse(wide, wide)
    r, h = ftb.block_norm(x[:0], x[:0], pre_weight=w)
    assert r.shape == (0, 64) and h.shape == (0, 64)


# ---- rotary positions ----
def ref_rope(x, positions, table, sections, order, pairs):
    half = table.shape[1] // 2
    if positions.dim() == 1:
        positions = positions[None]
    axes = positions.shape[0]
    sections = sections or (half,)
    axis, left = [], list(sections)
    for i in range(half):
        if order == "blocks":
            a = next(j for j in range(axes) if left[j])
            left[a] -= 1
        else:
            a = i % axes if i // axes < sections[i % axes] else 0
        axis.append(a)
    out, mag = x.double().clone(), x.double().abs()
    for i, a in enumerate(axis):
        p = positions[a].long()
        c, s = (table[p, j].double()[:, None] for j in (i, half + i))
        e0, e1 = (i, i + half) if pairs == "half" else (2 * i, 2 * i + 1)
        u, v = x[..., e0].double(), x[..., e1].double()
        out[..., e0], out[..., e1] = u * c - v * s, v * c + u * s
        mag[..., e0] = mag[..., e1] = u.abs() + v.abs()
    return out, 2.0 ** -22 * mag


def rope_case(tokens, Hq, Hkv, D, rot, dtype=BF, axes=1, order="blocks", pairs="half", page=16,
              sections=None, layout="nhd", pos=torch.int32, slot=torch.int64, fused=True, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    qkv = torch.randn(tokens, Hq + 2 * Hkv, D, generator=g, device="cuda").to(dtype)
    q, k, v = qkv.split([Hq, Hkv, Hkv], 1)
    if not fused:
        q, k, v = (t.contiguous() for t in (q, k, v))
    table = ftb.rope_table(500, rot)
    shape = (tokens,) if axes == 1 else (axes, tokens)
    positions = torch.randint(0, 500, shape, generator=g, device="cuda", dtype=pos)
    pages = tokens // page + 3
    caches = [torch.zeros(pages, page, Hkv, D, dtype=dtype, device="cuda") for _ in range(2)]
    if layout == "hnd":
        caches = [torch.zeros(pages, Hkv, page, D, dtype=dtype, device="cuda").transpose(1, 2)
                  for _ in range(2)]
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:tokens].to(slot)
    if tokens > 2:
        slots[1] = -1
    out = ftb.rope_append(q, k, v, positions, table, *caches, slots, sections=sections,
                          order=order, pairs=pairs)
    near(out, *ref_rope(q, positions, table, sections, order, pairs))
    keep = slots >= 0
    kr, kb = ref_rope(k, positions, table, sections, order, pairs)
    at = slots[keep].long()
    near(caches[0][at // page, at % page], kr[keep], kb[keep])
    assert torch.equal(caches[1][at // page, at % page], v[keep])
    for c, t in zip(caches, (k, v)):  # nothing else was written
        rest = c.clone()
        rest[at // page, at % page] = 0
        assert (rest == 0).all()
    q2, k2 = ftb.rope(q, k, positions, table, sections=sections, order=order, pairs=pairs)
    assert torch.equal(q2, out) and torch.equal(k2[keep], caches[0][at // page, at % page])


@pytest.mark.parametrize("pairs", ["half", "adjacent"])
@pytest.mark.parametrize("D,rot", [(128, 128), (64, 64), (80, 80), (80, 40), (96, 48), (128, 64),
                                   (66, 22), (2, 2), (256, 256), (512, 2)])
def test_rope_shapes(D, rot, pairs):
    rope_case(37, 6, 2, D, rot, pairs=pairs)


@pytest.mark.parametrize("order", ["blocks", "cyclic"])
@pytest.mark.parametrize("pairs", ["half", "adjacent"])
@pytest.mark.parametrize("sections", [(24, 20, 20), (64, 0, 0), (0, 32, 32), (22, 21, 21),
                                      (0, 0, 64)])
def test_rope_axes(order, pairs, sections):
    rope_case(50, 4, 1, 128, 128, axes=3, sections=sections, order=order, pairs=pairs)
    rope_case(50, 4, 1, 128, 128, axes=3, sections=sections, order=order, pairs=pairs, dtype=F16,
              pos=torch.int64, slot=torch.int32, layout="hnd")


@pytest.mark.parametrize("tokens", [1, 2, 3, 1000])
@pytest.mark.parametrize("page", [1, 16, 48])
def test_rope_tokens(tokens, page):
    rope_case(tokens, 32, 8, 128, 128, page=page)
    rope_case(tokens, 3, 3, 72, 36, page=page, dtype=F16, fused=False)


def test_rope_positions_outside_the_table():
    q = torch.ones(3, 2, 64, dtype=BF, device="cuda")
    table = ftb.rope_table(10, 64)
    at = torch.tensor([9, 10, -1], dtype=torch.int32, device="cuda")
    out, k = ftb.rope(q, q, at, table)
    assert torch.isfinite(out[0]).all() and torch.isnan(out[1:]).all() and torch.isnan(k[1:]).all()


def test_rope_table_is_exact_to_32_bits():
    t = ftb.rope_table(200000, 16, 1e6, device="cpu")
    angle = 199999 * 1e6 ** (-torch.arange(0, 16, 2, dtype=torch.float64) / 16)
    assert torch.equal(t[-1], torch.cat([angle.cos(), angle.sin()]).float())


def test_rope_in_place_and_refusals():
    q = torch.randn(5, 4, 64, device="cuda").to(BF)
    k = torch.randn(5, 2, 64, device="cuda").to(BF)
    table = ftb.rope_table(64, 64)
    at = torch.arange(5, dtype=torch.int32, device="cuda")
    cache = torch.zeros(2, 16, 2, 64, dtype=BF, device="cuda")
    want, _ = ftb.rope(q, k, at, table)
    args = dict(q=q, k=k, v=k, positions=at, table=table, k_cache=cache, v_cache=cache.clone(),
                slots=at)

    def refuse(**kw):
        with pytest.raises((ValueError, ftb._lib.FtbError)):
            ftb.rope_append(**{**args, **kw})

    refuse(k=k[:3])
    refuse(v=k.half())
    refuse(positions=at[:2])
    refuse(positions=at.float())
    refuse(positions=torch.stack([at, at]))  # two axes without sections
    refuse(sections=(16, 16))
    refuse(table=table.double())
    refuse(table=ftb.rope_table(64, 66))
    refuse(k_cache=cache.half())
    refuse(k_cache=cache[..., :32])
    refuse(slots=at[:4])
    refuse(pairs="both")
    refuse(order="random")
    refuse(q_out=torch.empty(5, 4, 64, device="cuda"))
    got = ftb.rope_append(**{**args, "q_out": q})
    assert got is q and torch.equal(q, want)


@pytest.mark.parametrize("H", [9, 63, 257, 2041, 2042, 4099, 8185, 8190, 16377, 16383])
@pytest.mark.parametrize("rows", [3, 700])
def test_block_norm_odd_widths_with_gates(H, rows):
    """Rows that follow one another at a width that is no multiple of 8, and views of them that
    start off a 16-byte boundary."""
    run_norm(rows, H, BF, F32, "full")
    run_norm(rows, H, F16, F16, "channel", "sigmoid")
    run_norm(rows, H, BF, BF, "token", post=False)
    x = torch.randn(rows * H + 1, device="cuda").to(BF)[1:].view(rows, H)
    w = torch.ones(H, dtype=BF, device="cuda")
    _, _, ref, b = ref_norm(x, None, None, None, 1, w, 1e-6, None)
    near(ftb.rms_norm(x, w), ref, b)
