"""Operators for token sequences on the GPU, against their definitions in 64 bits (sequence_oracle.py, which derives the bounds)."""
import math

import pytest
import torch

import sequence_oracle as orc

import dl_templates_b200 as swa

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, F16, BF = torch.float32, torch.float16, torch.bfloat16


def randn(g, *shape, dtype=BF):
    return torch.randn(*shape, generator=g, dtype=torch.float32).to(dtype)


def gen(*seed):
    return torch.Generator().manual_seed(hash(seed) & 0x7FFFFFFF)


def lens_tensor(lens):
    return None if lens is None else torch.tensor(lens, dtype=torch.int32, device=DEV)


# B, Hq, Hkv, N, window, n_sink, d_qk, d_v, lens
ATTN = [
    (1, 1, 1, 1, 1, 0, 64, 64, None),                       # one token
    (1, 2, 1, 5, 3, 1, 64, 64, None),
    (2, 4, 2, 129, 1, 0, 64, 64, None),                     # a window of the token alone
    (1, 4, 2, 129, 1, 3, 64, 64, [128]),
    (2, 2, 2, 200, 64, 4, 64, 64, [200, 131]),
    (3, 4, 4, 130, 40, 7, 64, 64, [0, 1, 129]),             # empty and single-token sequences
    (2, 6, 2, 333, 100, 16, 80, 80, [333, 257]),            # heads in threes, a head dim that fills no tile
    (1, 3, 3, 300, 128, 5, 96, 64, None),                   # odd heads, keys wider than values
    (1, 2, 1, 700, 129, 130, 128, 128, None),               # sinks over two blocks, window one beyond a block
    (1, 8, 1, 390, 127, 1, 64, 128, None),                  # all heads on one key head
    (1, 5, 1, 520, 250, 33, 128, 64, [515]),
    (1, 2, 2, 1100, 2000, 9, 128, 128, None),               # a window longer than the sequence
    (1, 2, 1, 1000, 200, 1000, 64, 64, None),               # every token a sink
    (2, 2, 2, 257, 256, 0, 8, 16, [257, -4]),               # small heads; a negative length is none
    (1, 4, 2, 384, 130, 300, 128, 128, [300]),
    (1, 2, 1, 140, 50, 4, 20, 36, None),                    # head dims that are no multiple of 8
    (1, 2, 1, 90, 30, 4, 72, 200, None),                    # beyond the tensor-core kernels
]


def attn_case(case, dtype):
    B, Hq, Hkv, N, W, ns, d, dv, lens = case
    g = gen(*case[:8])
    t = dict(q=randn(g, B, Hq, N, d, dtype=dtype), k=randn(g, B, Hkv, N, d, dtype=dtype), v=randn(g, B, Hkv, N, dv, dtype=dtype),
             do=randn(g, B, Hq, N, dv, dtype=dtype))
    return t, d ** -0.5


def run_attn(t, lens, W, ns, scale):
    """Into outputs full of NaN: a row that nobody writes shows."""
    x = {n: t[n].to(DEV) for n in t}
    outs = [torch.full_like(x[n], float("nan")) for n in ("do", "q", "k", "v")]
    o, lse = swa.sink_swa_forward(x["q"], x["k"], x["v"], W, ns, scale, lens, out=outs[0])
    dq, dk, dv = swa.sink_swa_backward(x["q"], x["k"], x["v"], o, lse, x["do"], W, ns, scale, lens, out=tuple(outs[1:]))
    swa.check_status()
    return dict(o=o, lse=lse, dq=dq, dk=dk, dv=dv)


@pytest.mark.parametrize("dtype", [F32, F16, BF], ids=["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("case", ATTN, ids=str)
def test_attention(case, dtype):
    _, _, _, _, W, ns, _, _, lens = case
    t, scale = attn_case(case, dtype)
    want, bound = orc.attention(t["q"], t["k"], t["v"], lens, W, ns, scale, t["do"])
    got = run_attn(t, lens_tensor(lens), W, ns, scale)
    for n in want:
        orc.check(got[n], want[n], bound[n], f"{n}")


@pytest.mark.parametrize("dtype", [F32, BF], ids=["fp32", "bf16"])
def test_attention_as_an_autograd_function(dtype):
    case = (2, 4, 2, 150, 60, 3, 64, 64, [150, 99])
    t, scale = attn_case(case, dtype)
    lens = lens_tensor(case[-1])
    x = {n: t[n].to(DEV).requires_grad_() for n in ("q", "k", "v")}
    want = run_attn(t, lens, 60, 3, scale)
    for f in (swa.SinkSwa.apply, super(swa.SinkSwa, swa.SinkSwa).apply):          # native and general path
        o = f(x["q"], x["k"], x["v"], lens, 60, 3, scale)
        assert torch.equal(o, want["o"])
        grads = torch.autograd.grad(o, list(x.values()), t["do"].to(DEV))
        for a, n in zip(grads, ("dq", "dk", "dv")):
            assert torch.equal(a, want[n]), n
    # only some inputs want gradients; a broadcast gradient; an expanded input gets the sum
    o = swa.SinkSwa.apply(x["q"].detach(), x["k"], x["v"].detach(), lens, 60, 3, scale)
    o.sum().backward()
    val, bound = orc.attention(t["q"], t["k"], t["v"], case[-1], 60, 3, scale, torch.ones_like(t["do"]))
    orc.check(x["k"].grad, val["dk"], bound["dk"], "dk of a sum")
    k1 = t["k"][:, :1].to(DEV).requires_grad_()
    o = swa.SinkSwa.apply(x["q"].detach(), k1.expand(-1, 2, -1, -1), x["v"].detach(), None, 60, 3, scale)
    o.backward(t["do"].to(DEV))
    val, bound = orc.attention(t["q"], t["k"][:, :1].expand(-1, 2, -1, -1), t["v"], None, 60, 3, scale, t["do"])
    dk = val["dk"].sum(1, keepdim=True)                       # (torch's sum over the heads rounds once more)
    orc.check(k1.grad, dk, bound["dk"].sum(1, keepdim=True) + 2 * orc.HALF[dtype] * dk.abs(), "dk of an expanded key")
    with pytest.raises(RuntimeError, match="second"):
        o = swa.SinkSwa.apply(x["q"], x["k"], x["v"], lens, 60, 3, scale)
        torch.autograd.grad(o.sum(), x["q"], create_graph=True)


@pytest.mark.parametrize("dtype", [F32, BF], ids=["fp32", "bf16"])
def test_attention_of_strided_tensors(dtype):
    """A packed projection output, read in place; results into views of larger buffers, whose other elements stay."""
    B, Hq, Hkv, N, d, W, ns = 2, 4, 2, 200, 64, 70, 5
    g = gen(7)
    qkv = randn(g, B, N, Hq + 2 * Hkv, d, dtype=dtype).to(DEV)
    do = randn(g, B, N, Hq, d, dtype=dtype).to(DEV).permute(0, 2, 1, 3)
    q, k, v = qkv.permute(0, 2, 1, 3).split([Hq, Hkv, Hkv], 1)
    o_buf = torch.full((B, N, Hq, d + 8), 7.0, device=DEV, dtype=dtype)
    out = o_buf[..., :d].permute(0, 2, 1, 3)
    o, lse = swa.sink_swa_forward(q, k, v, W, ns, 0.125, out=out)
    assert o.data_ptr() == out.data_ptr() and bool((o_buf[..., d:] == 7).all())
    dqkv = torch.full_like(qkv, 7.0)
    outs = dqkv.permute(0, 2, 1, 3).split([Hq, Hkv, Hkv], 1)
    swa.sink_swa_backward(q, k, v, o, lse, do, W, ns, 0.125, out=tuple(outs))
    o2, lse2 = swa.sink_swa_forward(q.contiguous(), k.contiguous(), v.contiguous(), W, ns, 0.125)
    g2 = swa.sink_swa_backward(q.contiguous(), k.contiguous(), v.contiguous(), o2, lse2, do.contiguous(), W, ns, 0.125)
    assert torch.equal(o, o2) and torch.equal(lse, lse2)
    for a, b in zip(outs, g2):
        assert torch.equal(a, b)
    with pytest.raises(ValueError, match="share memory"):
        swa.sink_swa_forward(q, k, v, W, ns, 0.125, out=torch.empty(B, 1, N, d, device=DEV, dtype=dtype).expand(-1, Hq, -1, -1))


@pytest.mark.parametrize("bad", [float("inf"), float("nan"), float("-inf")])
@pytest.mark.parametrize("dtype", [F32, F16, BF], ids=["fp32", "fp16", "bf16"])
def test_infinities_stay_with_the_rows_that_see_them(dtype, bad):
    """One key and one value of a token that some rows of a tile see and others do not, and padding that holds nothing but NaN."""
    B, Hq, Hkv, N, W, ns, d = 2, 2, 1, 420, 100, 4, 64
    lens = [420, 300]
    t, scale = attn_case((B, Hq, Hkv, N, W, ns, d, d, lens), dtype)
    clean = run_attn(t, lens_tensor(lens), W, ns, scale)
    for n in t:
        t[n][1, :, 300:] = float("nan")
    padded = run_attn(t, lens_tensor(lens), W, ns, scale)
    for n in clean:
        assert torch.equal(clean[n][0], padded[n][0]) and bool(torch.isfinite(padded[n][1, :, :300].float()).all()), n
    want, bound = orc.attention(*(torch.nan_to_num(t[n]) for n in ("q", "k", "v")), lens, W, ns, scale, torch.nan_to_num(t["do"]))
    for n in want:
        orc.check(padded[n], want[n], bound[n], n)
    j = 205
    t["v"][0, 0, j, 3] = bad
    got = run_attn(t, lens_tensor(lens), W, ns, scale)
    sees = torch.zeros(N, dtype=torch.bool)
    sees[j:j + W] = True
    o = got["o"][0].float().cpu()
    assert not torch.isfinite(o[:, sees, 3]).any()
    assert torch.isfinite(o[:, ~sees]).all() and torch.isfinite(o[:, sees][..., :3]).all()
    ref = clean["o"][0].float().cpu()
    tol = 2 * bound["o"][0]
    assert bool(((o - ref).abs()[:, ~sees] <= tol[:, ~sees]).all())
    # gradients: the rows that see token j have no finite dP; keys that share no row with j keep theirs
    for n, near in (("dq", sees), ("dk", torch.arange(N).sub(j).abs() < W)):
        x = got[n][0].float().cpu()
        near = near | (torch.arange(N) < ns) if n == "dk" else near
        assert torch.isfinite(x[:, ~near]).all(), n
        assert bool(((x - clean[n][0].float().cpu()).abs()[:, ~near] <= 2 * bound[n][0][:, ~near]).all()), n


def test_large_scores_and_late_maxima():
    """Scores of hundreds, rows whose maximum comes in the last block they meet: the running maximum has to follow."""
    B, H, N, W, d = 1, 2, 600, 500, 64
    g = gen(3)
    q, k, v, do = (randn(g, B, H, N, d) for _ in range(4))
    for scale_up in (1.0, 30.0):
        k2 = k * scale_up
        k2[:, :, ::97] *= 4
        k2[:, :, 0] *= 3
        want, bound = orc.attention(q, k2, v, None, W, 1, d ** -0.5, do)
        got = run_attn(dict(q=q, k=k2, v=v, do=do), None, W, 1, d ** -0.5)
        for n in want:
            orc.check(got[n], want[n], bound[n], n)


@pytest.mark.parametrize("scale", [-0.3, 0.0])
def test_scales_of_any_sign(scale):
    case = (1, 2, 1, 150, 60, 3, 64, 64, None)
    t, _ = attn_case(case, BF)
    want, bound = orc.attention(t["q"], t["k"], t["v"], None, 60, 3, scale, t["do"])
    got = run_attn(t, None, 60, 3, scale)
    for n in want:
        orc.check(got[n], want[n], bound[n], n)


def test_results_repeat_bit_for_bit():
    case = (2, 8, 2, 900, 200, 70, 128, 128, [900, 611])
    t, scale = attn_case(case, BF)
    a, b = (run_attn(t, lens_tensor(case[-1]), 200, 70, scale) for _ in range(2))
    for n in a:
        assert torch.equal(a[n], b[n]), n


# ---- rotation --------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F32, F16, BF], ids=["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("B, Hq, Hkv, N, C, R", [(1, 1, 1, 1, 64, (32,)), (2, 4, 2, 77, 64, (8, 12, 12)), (1, 3, 1, 130, 128, (16, 24, 24)),
                                                   (2, 5, 5, 33, 80, (10, 10)), (1, 2, 1, 19, 37, (3, 5, 7, 2)), (3, 16, 4, 700, 96, (8, 8, 16)),
                                                   (1, 2, 2, 40, 30, (1,)), (1, 32, 8, 2000, 128, (64,))])
def test_rotation(B, Hq, Hkv, N, C, R, dtype):
    g = gen(B, N, C)
    q, k, dq, dk = (randn(g, B, h, N, C, dtype=dtype) for h in (Hq, Hkv, Hq, Hkv))
    rows = [11 + 5 * a for a in range(len(R))]
    tabs = [swa.make_cs_table(r, n) for r, n in zip(R, rows)]
    for shape in ((len(R), N), (B, len(R), N)):
        pos = torch.randint(-2, 30, shape, generator=g, dtype=torch.int32)          # some not rotated, some behind the table's end
        dpos, dtabs = pos.to(DEV), [t.to(DEV) for t in tabs]
        x = [t.to(DEV).requires_grad_() for t in (q, k)]
        y = swa.RotaryPEAxes.apply(*x, dpos, *dtabs)
        grads = torch.autograd.grad(y, x, (dq.to(DEV), dk.to(DEV)))
        for got, src, inv in (*((a, b, False) for a, b in zip(y, (q, k))), *((a, b, True) for a, b in zip(grads, (dq, dk)))):
            orc.check(got, orc.rotate(src, pos, tabs, inv), orc.rotate_bound(src, pos, tabs, dtype, inv), "rotation")
        assert torch.equal(x[0].detach().cpu(), q)
        one = swa.rope_axes_apply_to(x[0].detach(), dpos, dtabs)
        assert torch.equal(one, y[0])
        gq, = torch.autograd.grad(swa.RotaryPEAxes.apply(*x, dpos, *dtabs)[0], x[0], dq.to(DEV))       # one output used only
        assert torch.equal(gq, grads[0])
        z = super(swa.RotaryPEAxes, swa.RotaryPEAxes).apply(*x, dpos, *dtabs)
        assert torch.equal(z[1], y[1]) and torch.equal(torch.autograd.grad(z, x, (dq.to(DEV), dk.to(DEV)))[1], grads[1])


def test_rotation_of_views_and_agreement_with_two_axes():
    """Strided, misaligned and expanded inputs; with two axes of equal pairs the operator is RotaryPE2D."""
    g = gen(5)
    B, N, H, C = 2, 60, 6, 64
    packed = randn(g, B, N, H, C + 3).to(DEV)
    pos = torch.randint(-1, 8, (2, N), generator=g, dtype=torch.int32)
    tabs = [swa.make_cs_table(16, 8).to(DEV)] * 2
    q, k = packed[..., 1:C + 1].permute(0, 2, 1, 3).split([4, 2], 1)
    y = swa.RotaryPEAxes.apply(q, k, pos.to(DEV), *tabs)
    z = swa.RotaryPEAxes.apply(q.contiguous(), k.contiguous(), pos.to(DEV), *tabs)
    assert torch.equal(y[0], z[0]) and torch.equal(y[1], z[1])
    e = k[:, :1].expand(-1, 3, -1, -1)
    assert torch.equal(swa.rope_axes_apply_to(e, pos.to(DEV), tabs), z[1][:, :1].expand(-1, 3, -1, -1))
    idx = ((pos[0] << 16) | (pos[1] & 0xFFFF)).to(torch.int32).to(DEV)
    flat = q.contiguous().view(-1, N, C)
    assert torch.equal(z[0].view(-1, N, C), swa.rope2d_apply_to(flat, idx, *tabs))


def test_rotation_refuses():
    q = torch.zeros(2, 2, 6, 16, device=DEV)
    pos, tab = torch.zeros(1, 6, dtype=torch.int32, device=DEV), torch.zeros(4, 8, 2, device=DEV)
    f = swa.RotaryPEAxes.apply
    for bad, exc in ((lambda: f(q, q, pos), ValueError), (lambda: f(q, q, pos, tab, tab), ValueError), (lambda: f(q, q, pos.long(), tab), TypeError),
                     (lambda: f(q, q, pos[:, :5], tab), ValueError), (lambda: f(q, q[:, :, :5], pos, tab), ValueError),
                     (lambda: f(q, q.half(), pos, tab), TypeError), (lambda: f(q, q, pos.cpu(), tab), RuntimeError),
                     (lambda: f(q, q, pos, tab.cpu()), RuntimeError), (lambda: f(q, q, pos, tab.double()), TypeError),
                     (lambda: f(q, q, pos, torch.zeros(4, 9, 2, device=DEV)), RuntimeError), (lambda: f(q.double(), q.double(), pos, tab), TypeError),
                     (lambda: f(q, q, pos, tab.clone().requires_grad_()), RuntimeError),
                     (lambda: f(q[0], q[0], pos, tab), ValueError), (lambda: f(q, q, pos[None].expand(3, 1, 6), tab), ValueError)):
        with pytest.raises(exc):
            bad()


# ---- paged cache ------------------------------------------------------------------------------------------------------------
def make_cache(g, B, Hkv, page, max_pages, d, dv, dtype, token_major=False):
    n_pages = B * max_pages + 2
    shape = (lambda x: (n_pages, page, Hkv, x)) if token_major else (lambda x: (n_pages, Hkv, page, x))
    kc, vc = randn(g, *shape(d), dtype=dtype), randn(g, *shape(dv), dtype=dtype)
    if token_major:
        kc, vc = kc.permute(0, 2, 1, 3), vc.permute(0, 2, 1, 3)
    table = torch.randperm(n_pages, generator=g)[: B * max_pages].view(B, max_pages).to(torch.int32)
    return kc, vc, table


@pytest.mark.parametrize("dtype", [F32, F16, BF], ids=["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("B, Hq, Hkv, T, page, d, dv, R, rot", [(3, 4, 2, 1, 16, 64, 64, (8, 12, 12), True), (2, 2, 1, 45, 7, 128, 64, (16, 24, 24), True),
                                                                  (4, 8, 8, 5, 1, 32, 96, (16,), True), (2, 3, 3, 19, 100, 37, 21, (4, 2), True),
                                                                  (2, 4, 2, 33, 16, 64, 64, (8,), False)])
def test_append(B, Hq, Hkv, T, page, d, dv, R, rot, dtype):
    g = gen(B, T, page, d)
    max_pages = -(-(T + 60) // page)
    q, k, v = randn(g, B, Hq, T, d, dtype=dtype), randn(g, B, Hkv, T, d, dtype=dtype), randn(g, B, Hkv, T, dv, dtype=dtype)
    kc, vc, table = make_cache(g, B, Hkv, page, max_pages, d, dv, dtype, token_major=B == 2)
    fresh = torch.randint(0, T + 1, (B,), generator=g).int()
    fresh[0] = T
    lens = fresh + torch.randint(0, 60, (B,), generator=g).int()
    table[-1, max_pages // 2] = -1                         # pages that are no pages: written to by nobody
    table[0, 0] = kc.shape[0]
    pos = torch.randint(-1, 9, (B, len(R), T), generator=g, dtype=torch.int32) if rot else None
    tabs = [swa.make_cs_table(r, 9) for r in R] if rot else None
    kr = orc.rotate(k, pos, tabs) if rot else k.double()
    kb = orc.rotate_bound(k, pos, tabs, dtype) if rot else torch.zeros_like(kr)
    wk, wv, bound = kc.double(), vc.double(), torch.zeros_like(kc, dtype=torch.float64)
    for b in range(B):
        for t in range(int(fresh[b])):
            p = int(lens[b]) - int(fresh[b]) + t
            pg = int(table[b, p // page])
            if 0 <= pg < kc.shape[0]:
                wk[pg, :, p % page], wv[pg, :, p % page], bound[pg, :, p % page] = kr[b, :, t], v[b, :, t].double(), kb[b, :, t]
    dk_, dv_ = (torch.empty_strided(c.shape, c.stride(), dtype=dtype, device=DEV).copy_(c) for c in (kc, vc))
    args = (None if pos is None else pos.to(DEV), tabs and [t.to(DEV) for t in tabs], dk_, dv_, table.to(DEV), lens.to(DEV), fresh.to(DEV))
    version = dk_._version
    y = swa.kv_append_rope(q.to(DEV), k.to(DEV), v.to(DEV), *args)
    assert dk_._version > version
    orc.check(dk_, wk, bound, "k cache")
    assert torch.equal(dv_.double().cpu(), wv)
    if rot:
        orc.check(y, orc.rotate(q, pos, tabs), orc.rotate_bound(q, pos, tabs, dtype), "q")
    else:
        assert torch.equal(y.cpu(), q)
    assert swa.kv_append_rope(None, k.to(DEV), v.to(DEV), *args) is None
    orc.check(dk_, wk, bound, "k cache again")


# B, Hq, Hkv, page, max_pages, d, dv, window, n_sink, lens
DECODE = [
    (1, 1, 1, 16, 1, 64, 64, 1, 0, [1]),
    (3, 4, 2, 16, 4, 64, 64, 20, 4, [0, 1, 64]),
    (2, 8, 1, 7, 40, 128, 128, 100, 3, [280, 101]),
    (2, 32, 4, 64, 10, 128, 128, 10000, 0, [639, 63]),          # a window longer than the cache
    (3, 6, 2, 100, 5, 80, 96, 130, 17, [500, 147, 148]),
    (1, 20, 1, 1, 300, 64, 128, 64, 64, [300]),                 # pages of one token, twenty heads on one
    (1, 3, 1, 16, 20, 37, 21, 90, 5, [311]),                    # odd head dims
    (2, 48, 2, 32, 64, 128, 64, 1500, 1, [2047, 1501]),
    (1, 2, 2, 16, 4, 160, 256, 40, 2, [50]),
]


@pytest.mark.parametrize("dtype", [F32, F16, BF], ids=["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("case", DECODE, ids=str)
def test_decode(case, dtype):
    B, Hq, Hkv, page, max_pages, d, dv, W, ns, lens = case
    g = gen(*case[:9])
    kc, vc, table = make_cache(g, B, Hkv, page, max_pages, d, dv, dtype, token_major=Hq == 6)
    q = randn(g, B, Hq, 1, d, dtype=dtype)
    want, bound = torch.zeros(B, Hq, 1, dv, dtype=torch.float64), torch.zeros(B, Hq, 1, dv, dtype=torch.float64)
    seen = torch.zeros(kc.shape[0], page, dtype=torch.bool)
    for b, n in enumerate(lens):
        if n:
            at = torch.arange(n)
            pg, pl = table[b][at // page].long(), at % page
            k, v = kc[pg, :, pl].transpose(0, 1), vc[pg, :, pl].transpose(0, 1)
            want[b, :, 0], bound[b, :, 0] = orc.decode(q[b, :, 0], k, v, W, ns, d ** -0.5)
            keep = (at >= n - W) | (at < ns)
            seen[pg[keep], pl[keep]] = True
            for i in range(max_pages):                     # pages that nothing of is seen may be anything
                if not bool(keep[i * page:(i + 1) * page].any()):
                    table[b, i] = [-1, 1 << 30][i % 2]
        else:
            table[b] = -7
    kc.permute(0, 2, 1, 3)[~seen] = float("nan")
    vc.permute(0, 2, 1, 3)[~seen] = float("nan")
    dk_, dv_ = (torch.empty_strided(c.shape, c.stride(), dtype=dtype, device=DEV).copy_(c) for c in (kc, vc))
    n = torch.tensor(lens, dtype=torch.int32, device=DEV)
    o = swa.sink_swa_decode(q.to(DEV), dk_, dv_, table.to(DEV), n, W, ns, d ** -0.5)
    orc.check(o, want, bound, "o")
    buf = torch.full((B, Hq, 3, dv), 5.0, dtype=dtype, device=DEV)
    swa.sink_swa_decode(q.to(DEV), dk_, dv_, table.to(DEV), n, W, ns, d ** -0.5, out=buf[:, :, 1:2])
    assert torch.equal(buf[:, :, 1:2], o) and bool((buf[:, :, ::2] == 5).all())


def test_cache_calls_refuse():
    g = gen(1)
    kc, vc, table = (t.to(DEV) for t in make_cache(g, 2, 2, 16, 2, 64, 64, BF))
    q, k = randn(g, 2, 4, 1, 64).to(DEV), randn(g, 2, 2, 1, 64).to(DEV)
    n = torch.ones(2, dtype=torch.int32, device=DEV)
    d, a = swa.sink_swa_decode, swa.kv_append_rope
    for bad, exc in ((lambda: d(q.float(), kc, vc, table, n, 4, 0), TypeError), (lambda: d(q[:, :3], kc, vc, table, n, 4, 0), ValueError),
                     (lambda: d(q.expand(-1, -1, 2, -1), kc, vc, table, n, 4, 0), ValueError), (lambda: d(q, kc, vc, table.long(), n, 4, 0), TypeError),
                     (lambda: d(q, kc, vc, table[:1], n, 4, 0), ValueError), (lambda: d(q, kc, vc, table, n.long(), 4, 0), TypeError),
                     (lambda: d(q, kc, vc, table.cpu(), n, 4, 0), RuntimeError), (lambda: d(q, kc, vc, table, n, 0, 0), RuntimeError),
                     (lambda: d(q, kc[:, :, :8], vc, table, n, 4, 0), ValueError), (lambda: d(q.clone().requires_grad_(), kc, vc, table, n, 4, 0), RuntimeError),
                     (lambda: a(q, k, k[:, :1], None, None, kc, vc, table, n), ValueError), (lambda: a(q, k, k, None, None, kc.float(), vc, table, n), TypeError),
                     (lambda: a(q, k, k, None, (torch.zeros(4, 8, 2, device=DEV),), kc, vc, table, n), ValueError),
                     (lambda: a(q, k, k, None, None, kc, vc[:1].expand_as(vc), table, n), ValueError),
                     (lambda: a(q, k, k, None, None, kc, vc, table, n, n.cpu()), RuntimeError)):
        with pytest.raises(exc):
            bad()


def test_offsets_beyond_32_bits():
    """A cache and query tensors of more than 2^31 elements: what lies behind is what a small tensor of the same rows gives."""
    g = gen(21)
    Hkv, page, d, n = 8, 64, 128, 300
    n_pages = (1 << 31) // (Hkv * page * d) + 8
    kc, vc = (torch.zeros(n_pages, Hkv, page, d, dtype=BF, device=DEV) for _ in range(2))
    k, v, q = randn(g, 1, Hkv, n, d).to(DEV), randn(g, 1, Hkv, n, d).to(DEV), randn(g, 1, 16, 1, d).to(DEV)
    lens = torch.tensor([n], dtype=torch.int32, device=DEV)
    outs = []
    for cache, first in (((kc, vc), n_pages - 5), ((kc[:5].clone(), vc[:5].clone()), 0)):
        table = torch.arange(first, first + 5, dtype=torch.int32, device=DEV)[None]
        swa.kv_append_rope(None, k, v, None, None, *cache, table, lens)
        outs.append(swa.sink_swa_decode(q, *cache, table, lens, 200, 4, 0.1))
        assert torch.equal(cache[0][first:first + 4].transpose(0, 1).reshape(Hkv, -1, d), k[0, :, :256])
    assert torch.equal(*outs)
    del kc, vc, cache
    N, H = 1 << 17, 129                               # 129 heads of 2^24 elements
    q, do = (torch.zeros(1, H, N, d, dtype=BF, device=DEV) for _ in range(2))
    k, v = randn(g, 1, 1, N, d).to(DEV), randn(g, 1, 1, N, d).to(DEV)
    q[:, -1], do[:, -1] = randn(g, N, d).to(DEV), randn(g, N, d).to(DEV)
    o, lse = swa.sink_swa_forward(q, k, v, 60, 3, 0.1)
    o1, lse1 = swa.sink_swa_forward(q[:, -1:], k, v, 60, 3, 0.1)
    assert torch.equal(o[:, -1:], o1) and torch.equal(lse[:, -1:], lse1)
    dq, dk, dv = swa.sink_swa_backward(q, k, v, o, lse, do, 60, 3, 0.1)
    dq1, dk1, dv1 = swa.sink_swa_backward(q[:, -1:], k, v, o1, lse1, do[:, -1:], 60, 3, 0.1)
    # the other heads' dO is zero, and so is their dS (the block with the sinks is summed in other pieces, so in another order)
    assert torch.equal(dq[:, -1:], dq1) and torch.equal(dv[:, :, 128:], dv1[:, :, 128:]) and torch.equal(dk[:, :, 128:], dk1[:, :, 128:])
    assert bool(torch.isfinite(dk.float()).all()) and bool(torch.isfinite(dv.float()).all())
    x = swa.rope_axes_apply_to(q, torch.zeros(1, N, dtype=torch.int32, device=DEV), (swa.make_cs_table(64, 4, device=DEV),))
    assert torch.equal(x[:, -1], q[:, -1])
    swa.check_status()


def test_largest_sinks_and_one_token_windows():
    """1024 sinks over many blocks, windows of one token, more heads than one MMA tile of the decoding kernel has."""
    for case, dtype in (((1, 2, 1, 1500, 1, 1024, 64, 64, None), BF), ((1, 24, 1, 260, 33, 2, 64, 64, [259]), BF),
                        # blocks with sinks in fewer pieces than their length asks for, or in one: so many heads that the SMs are busy
                        ((2, 40, 40, 1030, 20, 1024, 8, 8, [1030, 1027]), BF), ((1, 150, 150, 700, 1, 4, 8, 8, None), BF),
                        ((1, 150, 150, 700, 1, 4, 8, 8, None), F32)):
        _, _, _, _, W, ns, _, _, lens = case
        t, scale = attn_case(case, dtype)
        want, bound = orc.attention(t["q"], t["k"], t["v"], lens, W, ns, scale, t["do"])
        got = run_attn(t, lens_tensor(lens), W, ns, scale)
        for n in want:
            orc.check(got[n], want[n], bound[n], n)


# ---- together -----------------------------------------------------------------------------------------------------------------
def test_prompt_and_steps_agree_with_the_whole_sequence():
    """Rotate and attend over a prompt, put it into the cache, then single steps captured into a CUDA graph and replayed: the steps' results are
    those of the same tokens attended as one sequence."""
    B, Hq, Hkv, d, W, ns, page, P, steps = 2, 8, 2, 64, 40, 4, 16, 70, 9
    g = gen(11)
    N = P + steps
    q, k, v = randn(g, B, Hq, N, d).to(DEV), randn(g, B, Hkv, N, d).to(DEV), randn(g, B, Hkv, N, d).to(DEV)
    rope = swa.RotaryPositionEncodingAxes((8, 12, 12), (N, 8, 8)).to(DEV)
    pos = torch.stack([torch.arange(N), torch.arange(N) % 8, torch.arange(N) // 8 % 8]).int().to(DEV)
    qr, kr = rope(q, k, pos)
    whole = swa.sink_swa_fwd(qr, kr, v, W, ns, d ** -0.5)
    kc, vc, table = make_cache(g, B, Hkv, page, -(-N // page), d, d, BF)
    kc, vc, table = kc.to(DEV), vc.to(DEV), table.to(DEV)
    lens = torch.full((B,), P, dtype=torch.int32, device=DEV)
    swa.kv_append_rope(None, k[:, :, :P], v[:, :, :P], pos[:, :P], rope.tables, kc, vc, table, lens)
    sq, sk, sv, sp = (t.clone() for t in (q[:, :, P:P + 1], k[:, :, P:P + 1], v[:, :, P:P + 1], pos[:, P:P + 1]))

    def step():
        y = swa.kv_append_rope(sq, sk, sv, sp, rope.tables, kc, vc, table, lens)
        return swa.sink_swa_decode(y, kc, vc, table, lens, W, ns, d ** -0.5)
    lens += 1
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        eager = step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for t in range(steps):
        for dst, src in ((sq, q), (sk, k), (sv, v)):
            dst.copy_(src[:, :, P + t:P + t + 1])
        sp.copy_(pos[:, P + t:P + t + 1])
        graph.replay()
        if t == 0:
            assert torch.equal(out, eager)
        want, bound = orc.attention(*(x.cpu() for x in (qr[:, :, :P + t + 1], kr[:, :, :P + t + 1], v[:, :, :P + t + 1])), None, W, ns, d ** -0.5)
        orc.check(out, want["o"][:, :, -1:], bound["o"][:, :, -1:], f"step {t}")
        orc.check(whole[:, :, P + t:P + t + 1], want["o"][:, :, -1:], bound["o"][:, :, -1:], f"whole, token {P + t}")
        lens += 1


def test_training_step_in_a_graph_and_two_graphs():
    """Rotation and attention with their gradients, eagerly and captured; two captured steps replayed in turn keep to themselves."""
    B, Hq, Hkv, N, d, W, ns = 1, 4, 2, 300, 64, 90, 6
    g = gen(13)
    rope = swa.RotaryPositionEncodingAxes((16, 8, 8), (N, 16, 16)).to(DEV)
    pos = torch.stack([torch.arange(N), torch.arange(N) % 16, torch.arange(N) // 16 % 16]).int().to(DEV)

    def inputs():
        return [randn(g, B, h, N, d).to(DEV).requires_grad_() for h in (Hq, Hkv, Hkv)], randn(g, B, Hq, N, d).to(DEV)

    def step(x, do):
        qr, kr = rope(x[0], x[1], pos)
        o = swa.SinkSwa.apply(qr, kr, x[2], None, W, ns, d ** -0.5)
        return (o.detach(), *torch.autograd.grad(o, x, do))
    sets = [inputs() for _ in range(2)]
    eager = []
    for x, do in sets:
        eager.append([t.clone() for t in step(x, do)])
    graphs = []
    for x, do in sets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(x, do)
        graphs.append((graph, out))
    for _ in range(2):
        for graph, _ in graphs:
            graph.replay()
    torch.cuda.synchronize()
    for (_, out), want in zip(graphs, eager):
        for a, b in zip(out, want):
            assert torch.equal(a, b)
    # a leaf whose eager graph is alive on another stream cannot be captured: refused before anything is launched
    x, do = sets[0]
    alive = swa.SinkSwa.apply(x[0], x[1], x[2], None, W, ns, 0.1)
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    with pytest.raises(RuntimeError, match="still alive"):
        with torch.cuda.graph(graph, stream=side):
            swa.SinkSwa.apply(x[0], x[1], x[2], None, W, ns, 0.1)
    assert alive.grad_fn is not None
    torch.cuda.synchronize()
    assert torch.equal(step(x, do)[0], eager[0][0])


def test_capture_beside_a_live_graph_of_an_upstream_leaf():
    """The leaf whose eager graph lives lies behind other operations: refused all the same; without that graph the capture works, on two
    streams of one capture too."""
    g = gen(14)
    w = randn(g, 1, 2, 200, 64).to(DEV).requires_grad_()
    k, v = (randn(g, 1, 2, 200, 64).to(DEV) for _ in range(2))
    rope = swa.RotaryPositionEncodingAxes((32,), (200,)).to(DEV)
    pos = torch.arange(200, dtype=torch.int32, device=DEV)[None]

    def loss():
        qr, kr = rope(w * 2, k, pos)
        return swa.SinkSwa.apply(qr, kr, v, None, 50, 4, 0.125)
    want, = torch.autograd.grad(loss(), w, torch.ones_like(k))
    alive = w * 2
    graph, stream, fork = torch.cuda.CUDAGraph(), torch.cuda.Stream(), torch.cuda.Stream()
    with pytest.raises(RuntimeError, match="still alive"):
        with torch.cuda.graph(graph, stream=stream):
            loss()
    del alive
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        scaled = w * 2                                           # w's accumulator belongs to the captured stream from here on
        fork.wait_stream(stream)
        with torch.cuda.stream(fork):
            qr, kr = rope(scaled, k, pos)
            o = swa.SinkSwa.apply(qr, kr, v, None, 50, 4, 0.125)
        stream.wait_stream(fork)
        got, = torch.autograd.grad(o, w, torch.ones_like(k))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want)


def test_outputs_share_no_memory_and_count_as_written():
    g = gen(15)
    q, k, v = (randn(g, 1, 2, 40, 64).to(DEV) for _ in range(3))
    o, lse = swa.sink_swa_forward(q, k, v, 9, 2, 0.125)
    both = torch.empty(2, *q.shape, device=DEV, dtype=q.dtype)
    grads = [torch.empty_like(q) for _ in range(3)]
    cache = [torch.zeros(3, 2, 16, 64, device=DEV, dtype=q.dtype) for _ in range(2)]
    table, lens = torch.arange(3, dtype=torch.int32, device=DEV)[None], torch.tensor([40], dtype=torch.int32, device=DEV)
    one = q[:, :, :1].contiguous()
    bad = [lambda: swa.sink_swa_forward(q, k, v, 9, 2, 0.125, out=q), lambda: swa.sink_swa_forward(q, k, v, 9, 2, 0.125, out=v.view(v.shape)),
           lambda: swa.sink_swa_backward(q, k, v, o, lse, o, 9, 2, 0.125, out=(grads[0], grads[1], grads[0])),
           lambda: swa.sink_swa_backward(q, k, v, o, lse, o, 9, 2, 0.125, out=(q, grads[1], grads[2])),
           lambda: swa.sink_swa_backward(q, k, v, o, lse, o, 9, 2, 0.125, out=(grads[0], both[0], both.view(-1)[64:64 + q.numel()].view_as(q))),
           lambda: swa.kv_append_rope(None, k, v, None, (), cache[0], cache[0], table, lens),
           lambda: swa.kv_append_rope(None, cache[0][:1], v[:, :, :16], None, (), *cache, table[:, :1], lens),
           lambda: swa.sink_swa_decode(one, *cache, table, lens, 9, 2, out=one)]
    for f in bad:
        with pytest.raises(ValueError, match="shares memory"):
            f()
    # interleaved views of one buffer, as of a fused projection, are fine
    packed = torch.empty(1, 40, 3, 2, 64, device=DEV, dtype=q.dtype)
    views = [packed[:, :, i].transpose(1, 2) for i in range(3)]
    want = swa.sink_swa_backward(q, k, v, o, lse, o, 9, 2, 0.125)
    for a, b in zip(swa.sink_swa_backward(q, k, v, o, lse, o, 9, 2, 0.125, out=views), want):
        assert torch.equal(a, b)
    # autograd learns that an output it had saved was overwritten
    x = torch.ones_like(q, requires_grad=True)
    y = torch.empty_like(q)
    z = (x * y).sum()
    swa.sink_swa_forward(q, k, v, 9, 2, 0.125, out=y)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.backward()


def test_other_stream():
    case = (1, 2, 1, 400, 100, 4, 64, 64, None)
    t, scale = attn_case(case, BF)
    want = run_attn(t, None, 100, 4, scale)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = run_attn(t, None, 100, 4, scale)
    s.synchronize()
    for n in want:
        assert torch.equal(want[n], got[n]), n
