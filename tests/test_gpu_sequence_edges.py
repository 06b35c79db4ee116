"""Operators for token sequences where a tensor's layout, its padding or an unusual value must not change what is computed or how: against
64-bit definitions (sequence_oracle.py), or bit for bit against the same call on plain tensors."""
import pytest
import torch

import sequence_oracle as orc
from test_gpu_sequence import BF, DEV, F16, F32, attn_case, gen, lens_tensor, randn, run_attn

import dl_templates_b200 as swa

pytestmark = pytest.mark.gpu
NAMES = ("q", "k", "v", "do")


def same_bits(a, b):
    """Equal, NaN in the same places included."""
    return torch.equal(torch.nan_to_num(a, nan=1e4), torch.nan_to_num(b, nan=1e4)) and torch.equal(torch.isnan(a), torch.isnan(b))


# ---- padding -----------------------------------------------------------------------------------------------------------
# B, Hq, Hkv, N, window, n_sink, d_qk, d_v, lens: ends inside a block, at its first and last row, in the block of the sinks, before it
PADDED = [
    (2, 4, 2, 420, 100, 4, 64, 64, [300, 420]),
    (4, 2, 2, 400, 300, 16, 128, 128, [129, 255, 256, 257]),
    (2, 4, 1, 700, 90, 40, 128, 128, [651, 30]),            # pieces of the sinks' blocks; an end among the sinks
    (2, 3, 3, 500, 130, 130, 96, 64, [385, 131]),
    (1, 4, 2, 520, 200, 3, 64, 128, [401]),
    (3, 2, 1, 333, 64, 5, 80, 80, [1, 300, 0]),
    (1, 12, 4, 1500, 512, 16, 80, 80, [1033]),
]


@pytest.mark.parametrize("fill", [float("nan"), float("inf")])
@pytest.mark.parametrize("dtype", [F32, F16, BF], ids=["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("case", PADDED, ids=str)
def test_padding_that_is_not_finite_changes_no_bit(case, dtype, fill):
    """What lies behind a sequence's end takes no part: results are those of zeros there, bit for bit, so that no row is done a second time
    for it either."""
    _, _, _, N, W, ns, _, _, lens = case
    t, scale = attn_case(case, dtype)
    for value in (0.0, fill):
        for b, n in enumerate(lens):
            for x in NAMES:
                t[x][b, :, n:] = value
        got = run_attn(t, lens_tensor(lens), W, ns, scale)
        if value == 0.0:
            want = got
    for n in want:
        assert bool(torch.isfinite(got[n]).all()) or n == "lse", n
        assert torch.equal(got[n], want[n]), n


# ---- infinities ----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("d, dv", [(128, 128), (64, 64), (64, 128), (96, 40)])
@pytest.mark.parametrize("dtype", [F32, F16, BF], ids=["fp32", "fp16", "bf16"])
def test_an_infinity_in_one_piece_of_the_sinks_queries(dtype, d, dv):
    """One element of one query's dO, which shares a piece with queries that are finite: of the keys that see the query dK is lost, and one column
    of dV; all else stays what it is, and everything is the same bits on every run."""
    N, W, ns, i, c = 2000, 100, 70, 1500, 3
    t, scale = attn_case((1, 4, 1, N, W, ns, d, dv, None), dtype)
    want, bound = orc.attention(t["q"], t["k"], t["v"], None, W, ns, scale, t["do"])
    t["do"][0, 1, i, c] = float("inf")
    runs = [run_attn(t, None, W, ns, scale) for _ in range(4)]
    for r in runs[1:]:
        for n in r:
            assert same_bits(r[n], runs[0][n]), n
    got = {n: x.double().cpu() for n, x in runs[0].items()}
    j = torch.arange(N)
    sees = (j <= i) & ((j > i - W) | (j < ns))
    inside = lambda n, at: bool(((got[n] - want[n]).abs() <= bound[n])[at].all())
    columns = torch.arange(dv) != c
    assert not torch.isfinite(got["dk"][0, 0, sees]).any() and inside("dk", (0, 0, ~sees))
    assert not torch.isfinite(got["dv"][0, 0, sees, c]).any()
    assert inside("dv", (0, 0, ~sees)) and inside("dv", (0, 0, slice(None), columns))
    rows = torch.ones(4, N, dtype=torch.bool)
    rows[1, i] = False
    assert inside("dq", (0, rows)) and not torch.isfinite(got["dq"][0, 1, i]).all() and inside("o", (0,))


# ---- layouts -----------------------------------------------------------------------------------------------------------
def off_boundary(x):
    """The same values, contiguous, one element behind a 16-byte boundary."""
    y = torch.empty(x.numel() + 16, dtype=x.dtype, device=x.device)[1:1 + x.numel()].view(x.shape)
    return y.copy_(x)


def odd_rows(x):
    """The same values in rows that are five elements longer."""
    y = torch.empty(*x.shape[:3], x.shape[3] + 5, dtype=x.dtype, device=x.device)[..., :x.shape[3]]
    return y.copy_(x)


def reversed_dims(x):
    """The same values with heads and columns the other way round in memory."""
    return x.permute(3, 2, 0, 1).contiguous().permute(2, 3, 1, 0)


LAYOUTS = dict(off_boundary=off_boundary, odd_rows=odd_rows, reversed_dims=reversed_dims)


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("dtype", [F32, F16, BF], ids=["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("d, dv", [(64, 64), (128, 80)])
def test_layouts_of_inputs_and_outputs_change_no_bit(d, dv, dtype, layout):
    """Inputs or outputs that the tiled kernels cannot read or write in place are copied: the same kernels, the same bits.  One tensor at a
    time, then all."""
    f = LAYOUTS[layout]
    W, ns, lens = 70, 20, lens_tensor([333, 150])
    t, scale = attn_case((2, 4, 2, 333, W, ns, d, dv, None), dtype)
    x = {n: t[n].to(DEV) for n in NAMES}
    o, lse = swa.sink_swa_forward(x["q"], x["k"], x["v"], W, ns, scale, lens)
    want = swa.sink_swa_backward(x["q"], x["k"], x["v"], o, lse, x["do"], W, ns, scale, lens)
    for moved in [(n,) for n in (*NAMES, "out")] + [(*NAMES, "out")]:
        y = {n: f(x[n]) if n in moved else x[n] for n in NAMES}
        outs = [f(torch.full_like(z, 7.0)) if "out" in moved else torch.full_like(z, 7.0) for z in (o, *want)]
        o2, lse2 = swa.sink_swa_forward(y["q"], y["k"], y["v"], W, ns, scale, lens, out=outs[0])
        assert o2.data_ptr() == outs[0].data_ptr() and torch.equal(o2, o) and torch.equal(lse2, lse), moved
        o_in = f(o) if len(moved) > 1 else o
        got = swa.sink_swa_backward(y["q"], y["k"], y["v"], o_in, lse, y["do"], W, ns, scale, lens, out=tuple(outs[1:]))
        for a, b, z in zip(got, want, outs[1:]):
            assert a.data_ptr() == z.data_ptr() and torch.equal(a, b), moved
    swa.check_status()


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("dtype", [F32, F16, BF], ids=["fp32", "fp16", "bf16"])
def test_layouts_of_a_decoded_query_change_no_bit(dtype, layout):
    B, Hq, Hkv, page, n, d = 2, 8, 2, 16, 600, 64
    g = gen(61)
    kc, vc = (randn(g, 2 * n // page + 2, Hkv, page, d, dtype=dtype).to(DEV) for _ in range(2))
    q = randn(g, B, Hq, 1, d, dtype=dtype).to(DEV)
    table = torch.arange(2 * (n // page + 1), dtype=torch.int32, device=DEV).view(B, -1)
    lens = lens_tensor([n, n - 77])
    want = swa.sink_swa_decode(q, kc, vc, table, lens, 400, 4, 0.125)
    out = LAYOUTS[layout](torch.full_like(q, 7.0))
    got = swa.sink_swa_decode(LAYOUTS[layout](q), kc, vc, table, lens, 400, 4, 0.125, out=out)
    assert got.data_ptr() == out.data_ptr() and torch.equal(got, want)


@pytest.mark.parametrize("dtype", [F32, BF], ids=["fp32", "bf16"])
def test_gradient_of_a_sum_is_that_of_its_contiguous_copy(dtype):
    """o.sum() hands an expanded gradient on, all of whose strides are 0."""
    t, scale = attn_case((2, 4, 2, 500, 90, 4, 64, 64, None), dtype)
    x = [t[n].to(DEV).requires_grad_() for n in ("q", "k", "v")]
    want = torch.autograd.grad(swa.SinkSwa.apply(*x, None, 90, 4, scale), x, torch.ones_like(t["do"]).to(DEV))
    got = torch.autograd.grad(swa.SinkSwa.apply(*x, None, 90, 4, scale).sum(), x)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("d, dv", [(37, 21), (64, 90), (126, 128)])
def test_fp32_head_dims_that_fill_no_unit_are_padded(d, dv):
    """fp32 heads that are no multiple of 4: the tiled kernels' results with zero columns, bit for bit, and right."""
    case = (2, 4, 2, 300, 80, 6, d, dv, [300, 177])
    t, scale = attn_case(case, F32)
    pad = lambda z, n: torch.nn.functional.pad(z, (0, n - z.shape[3]))
    up = lambda n: (n + 3) // 4 * 4
    p = dict(q=pad(t["q"], up(d)), k=pad(t["k"], up(d)), v=pad(t["v"], up(dv)), do=pad(t["do"], up(dv)))
    want, got = (run_attn(z, lens_tensor(case[-1]), 80, 6, scale) for z in (p, t))
    val, bound = orc.attention(t["q"], t["k"], t["v"], case[-1], 80, 6, scale, t["do"])
    for n in got:
        assert torch.equal(got[n], want[n][..., :got[n].shape[-1]] if n != "lse" else want[n]), n
        orc.check(got[n], val[n], bound[n], n)


# ---- many heads --------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype, dv", [(F32, 132), (F32, 18), (F16, 9)], ids=str)
def test_backward_takes_as_many_heads_as_forward(dtype, dv):
    """More than 65535 heads in a batch, in layouts for every delta kernel: the gradients of each half of the batch."""
    B, H, Hkv, N, d = 2, 33000, 1000, 3, 4
    g = gen(B, H, dv)
    q, k, v, do = (randn(g, B, h, N, n, dtype=dtype).to(DEV) for h, n in ((H, d), (Hkv, d), (Hkv, dv), (H, dv)))
    for f in (lambda z: z, reversed_dims):
        for impl in ("auto", "simt"):
            o, lse = swa.sink_swa_forward(q, k, v, 2, 1, 0.5, impl=impl)
            got = swa.sink_swa_backward(q, k, v, o, lse, f(do), 2, 1, 0.5, impl=impl)
            for b in range(B):
                s = slice(b, b + 1)
                want = swa.sink_swa_backward(q[s], k[s], v[s], o[s], lse[s], f(do[s]), 2, 1, 0.5, impl=impl)
                for a, z in zip(got, want):
                    assert torch.equal(a[s], z)
    swa.check_status()


# ---- captures ----------------------------------------------------------------------------------------------------------
def test_a_whole_step_is_captured_after_a_warm_up_on_a_side_stream():
    """The usual recipe: some steps on a side stream, whose last loss (and with it the leaves' accumulators of that stream) stays alive, then the
    same step captured and replayed."""
    g = gen(31)
    N, W, ns = 200, 50, 4
    w = randn(g, 1, 2, N, 64).to(DEV).requires_grad_()
    k, v, do = (randn(g, 1, 2, N, 64).to(DEV) for _ in range(3))
    rope = swa.RotaryPositionEncodingAxes((32,), (N,)).to(DEV)
    pos = torch.arange(N, dtype=torch.int32, device=DEV)[None]

    def loss_of():
        qr, kr = rope(w * 2, k, pos)
        return (swa.SinkSwa.apply(qr, kr, v, None, W, ns, 0.125).float() * do.float()).sum()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(3):
            w.grad = None
            loss = loss_of()
            loss.backward()
    torch.cuda.current_stream().wait_stream(s)
    want = w.grad.clone()
    w.grad = None
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = loss_of()
        captured.backward()
    w.grad.fill_(float("nan"))
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(w.grad, want) and torch.equal(captured.detach(), loss.detach())
    swa.check_status()


# ---- entries without an autograd.Function ------------------------------------------------------------------------------
def raw_entries():
    g = gen(41)
    q, k, v = (randn(g, 1, 2, 40, 64).to(DEV) for _ in range(3))
    one = q[:, :, :1].contiguous()
    o, lse = swa.sink_swa_forward(q, k, v, 9, 2, 0.125)
    pos, tab = torch.zeros(1, 40, dtype=torch.int32, device=DEV), swa.make_cs_table(16, 8, device=DEV)
    kc, vc = (torch.zeros(3, 2, 16, 64, device=DEV, dtype=BF) for _ in range(2))
    table, lens = torch.arange(3, dtype=torch.int32, device=DEV)[None], torch.tensor([40], dtype=torch.int32, device=DEV)
    return {"sink_swa_fwd": (lambda x: swa.sink_swa_fwd(x, k, v, 9, 2, 0.125), q),
            "sink_swa_forward": (lambda x: swa.sink_swa_forward(q, x, v, 9, 2, 0.125)[0], k),
            "sink_swa_backward": (lambda x: swa.sink_swa_backward(q, k, v, o, lse, x, 9, 2, 0.125)[0], o),
            "rope_axes_apply_to": (lambda x: swa.rope_axes_apply_to(x, pos, (tab,)), q),
            "kv_append_rope": (lambda x: swa.kv_append_rope(x, k, v, None, None, kc, vc, table, lens), q),
            "sink_swa_decode": (lambda x: swa.sink_swa_decode(x, kc, vc, table, lens, 9, 2), one)}


@pytest.mark.parametrize("entry", ["sink_swa_fwd", "sink_swa_forward", "sink_swa_backward", "rope_axes_apply_to", "kv_append_rope", "sink_swa_decode"])
def test_entries_that_record_nothing_refuse_tangents_and_traces(entry):
    """A tangent would be dropped without a word, and a trace would hold an empty output and not the call."""
    import torch.autograd.forward_ad as fwAD
    f, x = raw_entries()[entry]
    with torch.no_grad():
        want = f(x).clone()
        with fwAD.dual_level():
            with pytest.raises(RuntimeError, match="tangent"):
                f(fwAD.make_dual(x, torch.ones_like(x)))
            assert torch.equal(f(x), want)                       # others go on
        with pytest.raises(RuntimeError, match="trace"):
            torch.jit.trace(f, (x,), check_trace=False)
        assert torch.equal(f(x), want)


# ---- as torch's autograd sees them ---------------------------------------------------------------------------------------
def functions():
    g = gen(43)
    q, k, v = randn(g, 2, 4, 90, 64).to(DEV), randn(g, 2, 2, 90, 64).to(DEV), randn(g, 2, 2, 90, 64).to(DEV)
    pos, tab = torch.arange(90, dtype=torch.int32, device=DEV)[None], swa.make_cs_table(16, 90, device=DEV)
    lens = lens_tensor([90, 51])
    return {"sink": lambda a, b, c: swa.SinkSwa.apply(a, b, c, lens, 30, 4, 0.125),
            "rope": lambda a, b, c: torch.cat(swa.RotaryPEAxes.apply(a, b, pos, tab), 1)}, (q, k, v)


@pytest.mark.parametrize("entry", ["sink", "rope"])
def test_forward_mode_and_functorch_are_refused(entry):
    import torch.autograd.forward_ad as fwAD
    fs, (q, k, v) = functions()
    f = fs[entry]
    for grad_mode in (True, False):
        with torch.set_grad_enabled(grad_mode), fwAD.dual_level():
            with pytest.raises((RuntimeError, NotImplementedError)):
                f(fwAD.make_dual(q, torch.ones_like(q)), k, v)
    with pytest.raises((RuntimeError, NotImplementedError)):
        torch.func.jvp(lambda x: f(x, k, v), (q,), (torch.ones_like(q),))
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda x: f(x, k, v).float().sum())(q)
    with pytest.raises(RuntimeError):
        torch.vmap(lambda x: f(x, k, v))(torch.stack([q, q]))


@pytest.mark.parametrize("entry", ["sink", "rope"])
def test_a_trace_holds_the_call_and_not_its_result(entry):
    fs, (q, k, v) = functions()
    f = fs[entry]
    with torch.no_grad():
        traced = torch.jit.trace(f, (q, k, v), check_trace=False)
        assert torch.equal(traced(q * 2, k * 3, v + 1), f(q * 2, k * 3, v + 1))


@pytest.mark.parametrize("entry", ["sink", "rope"])
def test_saved_tensor_hooks_and_checkpointing(entry):
    from torch.utils.checkpoint import checkpoint
    fs, ins = functions()
    f = fs[entry]
    ins = ins if entry == "sink" else ins[:2]
    call = f if entry == "sink" else lambda a, b: f(a, b, None)
    res = []
    for wrap in (lambda *t: call(*t), lambda *t: checkpoint(call, *t, use_reentrant=False), lambda *t: checkpoint(call, *t, use_reentrant=True)):
        t = [x.clone().requires_grad_(True) for x in ins]
        o = wrap(*t)
        o.float().square().sum().backward()
        res.append([o.detach(), *(x.grad for x in t)])
    packs = []
    with torch.autograd.graph.saved_tensors_hooks(lambda x: (packs.append(1), x.cpu())[1], lambda x: x.to(DEV)):
        t = [x.clone().requires_grad_(True) for x in ins]
        o = call(*t)
    o.float().square().sum().backward()
    res.append([o.detach(), *(x.grad for x in t)])
    assert len(packs) >= 2
    for r in res[1:]:
        assert all(torch.equal(a, b) for a, b in zip(r, res[0]))


# ---- threads, streams ----------------------------------------------------------------------------------------------------
def attn_step(t, lens, W, ns, scale):
    x = [t[n].detach().requires_grad_(True) for n in ("q", "k", "v")]
    pos = torch.arange(t["q"].shape[2], dtype=torch.int32, device=DEV)[None]
    tab = swa.make_cs_table(4, 64, device=DEV)
    qr, kr = swa.RotaryPEAxes.apply(x[0], x[1], pos, tab)
    o = swa.SinkSwa.apply(qr, kr, x[2], lens, W, ns, scale)
    return (o.detach(), *torch.autograd.grad(o, x, t["do"]))


def test_two_threads_on_two_streams():
    import threading
    cases = []
    for c, dtype in (((2, 4, 2, 400, 100, 16, 64, 64, [400, 333]), BF), ((1, 2, 1, 500, 60, 130, 128, 128, None), F16),
                     ((1, 4, 4, 210, 50, 4, 32, 32, [200]), F32), ((1, 3, 3, 300, 128, 5, 96, 64, None), BF)):
        t, scale = attn_case(c, dtype)
        cases.append(({n: z.to(DEV) for n, z in t.items()}, lens_tensor(c[-1]), c[4], c[5], scale))
    torch.cuda.synchronize()
    results, errors = [[], []], []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for r in range(10):
                    for j in range(len(cases)):
                        c = (j * (2 * i + 1) + r) % len(cases)
                        results[i].append((c, attn_step(*cases[c])))
                torch.cuda.current_stream().synchronize()
        except Exception as e:                               # noqa: BLE001 (shown by the assertion below)
            errors.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not errors
    torch.cuda.synchronize()
    swa.check_status()
    want = [attn_step(*c) for c in cases]
    for per_thread in results:
        assert len(per_thread) == 40
        for c, got in per_thread:
            assert all(torch.equal(a, b) for a, b in zip(got, want[c]))


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
def test_kernels_started_early_between_foreign_ones(dtype):
    """Products write the inputs right before the calls, and they are overwritten right after: training step, then append and decode."""
    W, ns = 90, 4
    sets = []
    for s in range(3):
        g = gen(51, s)
        sets.append({n: randn(g, 1, h, 700, 64, dtype=dtype).to(DEV) for n, h in (("q", 4), ("k", 2), ("v", 2), ("do", 4))})
    eye = torch.eye(64, device=DEV, dtype=dtype)
    kc, vc = (torch.zeros(12, 2, 64, 64, device=DEV, dtype=dtype) for _ in range(2))
    table, lens = torch.arange(12, dtype=torch.int32, device=DEV)[None], torch.tensor([700], dtype=torch.int32, device=DEV)
    live = {n: torch.empty_like(x) for n, x in sets[0].items()}

    def sequence(src):
        for n in live:
            torch.matmul(src[n], eye, out=live[n])
        got = attn_step(live, None, W, ns, 0.125)
        swa.kv_append_rope(None, live["k"], live["v"], None, None, kc, vc, table, lens)
        o = swa.sink_swa_decode(live["q"][:, :, -1:], kc, vc, table, lens, W, ns, 0.125)
        for x in (*live.values(), kc, vc):
            x.fill_(float("nan"))
        return (*got, o)
    prev = torch.backends.cuda.matmul.allow_tf32
    torch.backends.cuda.matmul.allow_tf32 = False
    try:
        want = []
        for s in sets:
            want.append([x.clone() for x in sequence(s)])
            torch.cuda.synchronize()
        with torch.cuda.stream(torch.cuda.Stream()):
            runs = [[sequence(s) for s in sets] for _ in range(4)]
            torch.cuda.current_stream().synchronize()
    finally:
        torch.backends.cuda.matmul.allow_tf32 = prev
    for got in runs:
        for a, b in zip(got, want):
            assert all(torch.equal(x, y) for x, y in zip(a, b))
    assert all(bool(torch.isfinite(x).all()) for x in want[0])
    swa.check_status()


# ---- widths of the blocks of sinks, wide heads ------------------------------------------------------------------------------
# B, Hq, Hkv, N, window, n_sink, d_qk, d_v, lens: blocks of sinks of 16 to 128 columns below the window, with P over the scores (d_v > 64) and beside
SINKS = [(1, 4, 2, 700, 100, ns, d, dv, None) for ns in (17, 40, 64, 100, 130, 200) for d, dv in ((128, 128), (64, 128), (64, 64))] + [
    (1, 3, 3, 900, 200, 70, 128, 128, [811]),
    (1, 3, 3, 600, 100, 90, 128, 64, [555]),
    (2, 2, 1, 400, 70, 9, 256, 256, [400, 288]),            # beyond the tensor-core kernels
    (1, 2, 2, 300, 64, 33, 136, 40, None),
]


@pytest.mark.parametrize("dtype", [F32, F16, BF], ids=["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("case", SINKS, ids=str)
def test_blocks_of_sinks_of_every_width(case, dtype):
    _, _, _, _, W, ns, _, _, lens = case
    t, scale = attn_case(case, dtype)
    want, bound = orc.attention(t["q"], t["k"], t["v"], lens, W, ns, scale, t["do"])
    got = run_attn(t, lens_tensor(lens), W, ns, scale)
    for n in want:
        orc.check(got[n], want[n], bound[n], n)


@pytest.mark.parametrize("bad", [float("inf"), float("nan"), float("-inf")])
@pytest.mark.parametrize("dtype", [F32, F16, BF], ids=["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("ns", [40, 130])
@pytest.mark.parametrize("d, dv", [(128, 128), (64, 128), (128, 64)])
def test_infinities_of_a_value_or_a_key(d, dv, ns, dtype, bad):
    """One element of a value: o loses one column of the rows that see it, dV nothing at all.  One element of a key: a row whose score with it is
    -inf goes on without it."""
    N, W, j, c = 420, 100, 205, 3
    t, scale = attn_case((1, 2, 1, N, W, ns, d, dv, None), dtype)
    want, bound = orc.attention(t["q"], t["k"], t["v"], None, W, ns, scale, t["do"])
    i = torch.arange(N)
    sees = (i >= j) & (i < j + W)
    inside = lambda got, n, at: bool(((got[n].double().cpu() - want[n]).abs() <= bound[n])[at].all())
    planted = {n: x.clone() for n, x in t.items()}
    planted["v"][0, 0, j, c] = bad
    got = run_attn(planted, None, W, ns, scale)
    others = torch.arange(dv) != c
    assert not torch.isfinite(got["o"][0][:, sees, c]).any()
    assert inside(got, "o", (0, slice(None), ~sees)) and inside(got, "o", (0, slice(None), slice(None), others))
    assert inside(got, "lse", (0,)) and inside(got, "dv", (0,)) and inside(got, "dq", (0, slice(None), ~sees))
    assert not torch.isfinite(got["dq"][0][:, sees]).all(-1).any()
    alone = ((i - j).abs() >= W) & (i >= ns)                 # keys that no row sees together with j
    assert inside(got, "dk", (0, slice(None), alone))
    planted = {n: x.clone() for n, x in t.items()}
    planted["k"][0, 0, j, c] = bad
    o = run_attn(planted, None, W, ns, scale)["o"].double().cpu()
    assert bool(((o - want["o"]).abs() <= bound["o"])[0][:, ~sees].all())
    minus = sees & (t["q"][0, :, :, c].double() * bad == float("-inf"))
    assert not torch.isfinite(o[0][sees & ~minus]).any()
    if bad == bad:
        # without key j: the same rows with a key that scores far below the others
        low = {n: x.double() for n, x in t.items()}
        see = orc.visible(N, W, ns, N)
        see[:, j] = False
        S = (low["q"][0] @ low["k"][0, 0].T * scale).masked_fill(~see, float("-inf"))
        ref = torch.softmax(S, -1) @ low["v"][0, 0]
        # (each weight is off by as much as in the row with key j, relative to itself)
        off = (ref.abs() + torch.softmax(S, -1) @ low["v"][0, 0].abs()) * (2 * orc.HALF[dtype] + 2.0 ** -16) + orc.floor_of(dtype) * N
        assert bool(((o[0] - ref).abs() <= off)[minus].all())
