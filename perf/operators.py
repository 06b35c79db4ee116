"""Timed cases of the operators for token sequences: rotary positions with several axes, attention with a sliding window and a
few first tokens that stay visible, and the paged cache that serves both (append with rotation, attention of single tokens).

A case is a plain dict; `op` says which operator:

  "rope"    RotaryPEAxes.apply: q and k rotated by positions on several axes (time, height, width)
  "attn"    SinkSwa.apply: token i sees the `window` latest tokens up to itself and the first `n_sink` ones
  "append"  kv_append_rope: new keys rotated into the pages of a cache, their values beside them, the queries rotated on the way
  "decode"  sink_swa_decode: one new token of each sequence attends over the cache

  train     forward and backward (gradients of every input) or forward only
  dtype     "bf16", "fp16" or "fp32"
  B, Hq, Hkv, N     batch, heads of queries and of keys (Hkv divides Hq), tokens ("append": new ones of a sequence)
  dqk, dv           head dims; r0, r1, r2: rotated pairs of each axis, 2 * (r0 + r1 + r2) <= dqk
  ragged            sequences of a batch have different lengths
  ctx, page         tokens of the longest sequence in the cache, tokens of a page
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
GRID = 64                      # positions of an image axis; the time axis is as long as the sequence


def _rope(name, train, dtype, B, Hq, Hkv, N, dqk, r0, r1, r2):
    return dict(name=name, op="rope", train=train, dtype=dtype, B=B, Hq=Hq, Hkv=Hkv, N=N, dqk=dqk, r0=r0, r1=r1, r2=r2)


def _attn(name, train, dtype, B, Hq, Hkv, N, window, n_sink, dqk, dv, ragged=False):
    return dict(name=name, op="attn", train=train, dtype=dtype, B=B, Hq=Hq, Hkv=Hkv, N=N, window=window, n_sink=n_sink,
                dqk=dqk, dv=dv, ragged=ragged)


def _append(name, dtype, B, Hq, Hkv, N, ctx, page, dqk, dv, r0, r1, r2, ragged=False):
    return dict(name=name, op="append", dtype=dtype, B=B, Hq=Hq, Hkv=Hkv, N=N, ctx=ctx, page=page, dqk=dqk, dv=dv,
                r0=r0, r1=r1, r2=r2, ragged=ragged)


def _decode(name, dtype, B, Hq, Hkv, ctx, page, window, n_sink, dqk, dv, ragged=False):
    return dict(name=name, op="decode", dtype=dtype, B=B, Hq=Hq, Hkv=Hkv, ctx=ctx, page=page, window=window, n_sink=n_sink,
                dqk=dqk, dv=dv, ragged=ragged)


def listed():
    return [
        # q and k of one image of 12 x 13 patches and a short caption, inference: a small call
        _rope("rope_infer_image", False, "fp16", 1, 8, 2, 173, 64, 8, 12, 12),
        # a training step's rotation over a video clip
        _rope("rope_train_video", True, "bf16", 2, 16, 4, 8192, 128, 16, 24, 24),
        # full precision, a part of the head rotated, odd number of tokens
        _rope("rope_train_part_fp32", True, "fp32", 2, 6, 3, 1999, 96, 8, 12, 4),
        # a short prompt through one layer: latency of a single call
        _attn("attn_infer_short", False, "bf16", 1, 8, 2, 200, 128, 4, 64, 64),
        # a padded training batch, head dim that fills no tile
        _attn("attn_train_padded", True, "fp16", 4, 12, 4, 1500, 512, 16, 80, 80, ragged=True),
        # full-precision training of a small model
        _attn("attn_train_fp32", True, "fp32", 2, 4, 4, 777, 256, 4, 64, 64),
        # long-context training, grouped heads
        _attn("attn_train_long", True, "bf16", 1, 16, 4, 16384, 1024, 64, 128, 128),
        # prefill of a long prompt with a wide window
        _attn("attn_prefill_long", False, "bf16", 1, 16, 4, 8192, 4096, 4, 128, 128),
        # one decoding step of a serving batch: one new token of each sequence
        _append("append_step", "bf16", 64, 32, 8, 1, 3000, 16, 128, 128, 16, 24, 24, ragged=True),
        # prompts of different lengths into the cache, q rotated beside
        _append("append_prompts", "fp16", 6, 16, 4, 2048, 4096, 64, 128, 128, 16, 24, 24, ragged=True),
        # one sequence being answered: latency
        _decode("decode_one", "bf16", 1, 32, 8, 5000, 64, 2048, 4, 128, 128),
        # a serving batch with a wide window
        _decode("decode_batch", "bf16", 64, 32, 8, 5000, 64, 4096, 4, 128, 128, ragged=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "attn", "attn", "attn", "append", "decode", "decode"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    Hkv = rng.choice([1, 2, 3, 4, 8])
    Hq = Hkv * rng.choice([1, 2, 3, 4, 6, 8])
    dqk = rng.choice([32, 64, 64, 80, 96, 128, 128])
    dv = rng.choice([dqk, dqk, 64, 128])
    r0, r1, r2 = rng.choice([(dqk // 8, dqk // 8 + dqk // 16, dqk // 8 + dqk // 16), (dqk // 8, dqk // 8, 0), (4, 4, 4)])
    ragged = rng.random() < 0.5
    if op == "rope":
        c = _rope("", rng.random() < 0.6, dtype, rng.randint(1, 4), Hq, Hkv, _log(rng, 33, 12000), dqk, r0, r1, r2)
        while c["B"] * c["N"] * (Hq + Hkv) * dqk > 42_000_000:
            c["N"] = c["N"] * 2 // 3
    elif op == "attn":
        N = _log(rng, 60, 12000)
        window = min(_log(rng, 32, 4096), N)
        c = _attn("", rng.random() < 0.6, dtype, rng.randint(1, 4), Hq, Hkv, N, window, rng.choice([0, 1, 4, 16, 64, 130]), dqk, dv,
                  ragged)
        most = 4.5e11 if dtype != "fp32" else 4.0e10
        while _work_attn(dict(c, train=True))["flops"] > most or c["B"] * Hq * c["N"] * min(2 * c["window"], c["N"]) > 600_000_000:
            c["N"] = max(32, c["N"] * 2 // 3)
            c["window"] = min(max(16, c["window"] * 4 // 5), c["N"])
    elif op == "append":
        N = rng.choice([1, 1, _log(rng, 2, 3000)])
        B = _log(rng, 1, 96) if N == 1 else rng.randint(1, 6)
        c = _append("", dtype, B, Hq, Hkv, N, N + _log(rng, 1, 3000), rng.choice([8, 16, 32, 64, 100]), dqk, dv, r0, r1, r2, ragged)
        while c["B"] * c["ctx"] * Hkv * (dqk + dv) > 150_000_000 or c["B"] * c["N"] * Hq * dqk > 30_000_000:
            c["B"] = max(1, c["B"] * 2 // 3)
            c["N"] = max(1, c["N"] * 3 // 4)
            c["ctx"] = max(c["N"] + 1, c["ctx"] * 3 // 4)
    else:
        ctx = _log(rng, 100, 9000)
        c = _decode("", dtype, _log(rng, 1, 64), Hq, Hkv, ctx, rng.choice([8, 16, 32, 64, 100]), _log(rng, 64, 6000),
                    rng.choice([0, 1, 4, 16, 64]), dqk, dv, ragged)
        while c["B"] * c["ctx"] * Hkv * (dqk + dv) * (2 if dtype == "fp32" else 1) > 300_000_000:
            c["B"] = max(1, c["B"] * 2 // 3)
            c["ctx"] = max(65, c["ctx"] * 4 // 5)
    del c["name"]
    return c


# ---- what a case's program has in hand ------------------------------------------------------------------------------------
def _lens(n_seq, longest, ragged):
    """Lengths of a batch's sequences: all the same, or spread evenly down to a third of the longest."""
    return [longest - (b * (2 * longest // 3)) // max(1, n_seq - 1) if ragged else longest for b in range(n_seq)]


def _table(n_pairs, n_pos, device):
    inv = 10000.0 ** (-torch.arange(n_pairs, dtype=torch.float64, device=device) / max(1, n_pairs))
    ang = torch.arange(n_pos, dtype=torch.float64, device=device)[:, None] * inv
    return torch.stack([ang.cos(), ang.sin()], -1).float().contiguous()


def _tables(case, n_time, device):
    return [_table(r, n, device) for r, n in ((case["r0"], n_time), (case["r1"], GRID), (case["r2"], GRID)) if r]


def _positions(case, B, T, first, g, dev):
    """[B, axes, T]: a text token moves on along the time axis and has no place in an image, an image's patches share the time."""
    axes = 1 + (case["r1"] > 0) + (case["r2"] > 0)
    t = torch.arange(T, device=dev) + first[:, None]
    cut = torch.randint(0, T + 1, (B, 1), generator=g, device=dev)
    text = torch.arange(T, device=dev) < cut
    w = 5 + int(torch.randint(0, 9, (1,), generator=g, device=dev))
    row, col = (t // w) % GRID, t % w
    p = torch.stack([t, torch.where(text, -1, row), torch.where(text, -1, col)][:axes], 1)
    return p.to(torch.int32).contiguous()


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=dev).to(dt)

    B, Hq, Hkv, dqk = case["B"], case["Hq"], case["Hkv"], case["dqk"]
    s = dict(case=dict(case))
    if case["op"] == "rope":
        N = case["N"]
        s["q"], s["k"] = randn(B, Hq, N, dqk), randn(B, Hkv, N, dqk)
        if case["train"]:
            s["dq"], s["dk"] = randn(B, Hq, N, dqk), randn(B, Hkv, N, dqk)
        s["pos"] = _positions(case, B, N, torch.zeros(B, dtype=torch.long, device=dev), g, dev)
        s["tables"] = _tables(case, N, dev)
        return s
    if case["op"] == "attn":
        N, dv = case["N"], case["dv"]
        s["q"], s["k"], s["v"] = randn(B, Hq, N, dqk), randn(B, Hkv, N, dqk), randn(B, Hkv, N, dv)
        if case["train"]:
            s["do"] = randn(B, Hq, N, dv)
        s["lens"] = torch.tensor(_lens(B, N, True), dtype=torch.int32, device=dev) if case["ragged"] else None
        s["sm_scale"] = dqk ** -0.5
        return s
    # a cache: pages in the order in which the sequences of a running server happened to ask for them
    dv, page, ctx = case["dv"], case["page"], case["ctx"]
    per_seq = -(-ctx // page)
    n_pages = B * per_seq + 1
    s["page_table"] = torch.randperm(n_pages, generator=g, device=dev)[: B * per_seq].to(torch.int32).reshape(B, per_seq)
    s["lens"] = torch.tensor(_lens(B, ctx, case["ragged"]), dtype=torch.int32, device=dev)
    s["k_cache"], s["v_cache"] = randn(n_pages, Hkv, page, dqk), randn(n_pages, Hkv, page, dv)
    if case["op"] == "append":
        T = case["N"]
        s["q"], s["k"], s["v"] = randn(B, Hq, T, dqk), randn(B, Hkv, T, dqk), randn(B, Hkv, T, dv)
        new = [min(n, l) for n, l in zip(_lens(B, T, case["ragged"] and T > 1), _lens(B, ctx, case["ragged"]))]
        s["new_lens"] = torch.tensor(new, dtype=torch.int32, device=dev)
        s["pos"] = _positions(case, B, T, (s["lens"] - s["new_lens"]).long(), g, dev)
        s["tables"] = _tables(case, ctx + T, dev)
    else:
        s["q"] = randn(B, Hq, 1, dqk)
        s["sm_scale"] = dqk ** -0.5
    return s


# ---- one pass ---------------------------------------------------------------------------------------------------------------
def _rotate(x, pos, tables, sign=1.0):
    """Pairs (i, i + R) of each axis' 2 R dims turned by the position's angle; a negative position turns nothing."""
    y, at = [], 0
    for a, tab in enumerate(tables):
        R = tab.shape[1]
        p = pos[:, a].long()
        cs = torch.where((p >= 0)[..., None, None], tab[p.clamp(min=0)], torch.tensor([1.0, 0.0], device=x.device))[:, None]
        u, w = x[..., at:at + R].float(), x[..., at + R:at + 2 * R].float()
        c, s = cs[..., 0], sign * cs[..., 1]
        y += [u * c - w * s, u * s + w * c]
        at += 2 * R
    return torch.cat(y + [x[..., at:].float()], -1).to(x.dtype)


def _banded(x, W, pad):
    """[.., N, d] as blocks of W rows with the block before beside each: [.., nb, 2 W, d] in 32 bits."""
    x = torch.nn.functional.pad(x.float(), (0, 0, 0, pad)).unflatten(-2, (-1, W))
    return torch.cat([torch.nn.functional.pad(x, (0, 0, 0, 0, 1, 0))[..., :-1, :, :], x], -2)


def _unbanded(x, N):
    """The transpose of _banded: the sum over the places where a row stands."""
    W = x.shape[-2] // 2
    before, own_block = x[..., :W, :], x[..., W:, :]
    return (own_block + torch.nn.functional.pad(before[..., 1:, :, :], (0, 0, 0, 0, 0, 1))).flatten(-3, -2)[..., :N, :]


def _plain_attn(s):
    c, q, k, v = s["case"], s["q"], s["k"], s["v"]
    B, Hq, N, _ = q.shape
    Hkv, G = k.shape[1], Hq // k.shape[1]
    W, ns, scale = min(c["window"], N), min(c["n_sink"], N), s["sm_scale"]
    pad = -N % W
    nb = (N + pad) // W
    length = s["lens"].view(B, 1, 1, 1) if s["lens"] is not None else torch.full((B, 1, 1, 1), N, device=q.device)

    def rows(x):                       # [B, Hq, N, d] -> [B, Hkv, nb, G W, d]
        x = torch.nn.functional.pad(x.float(), (0, 0, 0, pad)).view(B, Hkv, G, nb, W, -1)
        return x.transpose(2, 3).reshape(B, Hkv, nb, G * W, -1)

    def unrows(x):
        return x.view(B, Hkv, nb, G, W, -1).transpose(2, 3).reshape(B, Hq, nb * W, -1)[:, :, :N]

    i = torch.arange(nb * W, device=q.device).view(nb, 1, W, 1).expand(nb, G, W, 1).reshape(nb, G * W, 1)
    j = torch.arange(2 * W, device=q.device) + (torch.arange(nb, device=q.device)[:, None, None] - 1) * W
    live = i < length[..., None]                                          # [B, 1, nb, G W, 1]
    near = ((j <= i) & (j > i - W) & (j >= 0)) & (j < length[..., None]) & live
    js = torch.arange(ns, device=q.device)
    far = (js <= i - W) & (js < length[..., None]) & live
    # rows behind a sequence's end take no part, whatever they hold
    own_row = torch.arange(N, device=q.device).view(1, 1, N, 1) < length
    zero = torch.zeros((), device=q.device)
    q_, k_, v_ = (torch.where(own_row, x.float(), zero) for x in (q, k, v))
    qr, kb, vb = rows(q_), _banded(k_, W, pad), _banded(v_, W, pad)
    ks, vs = k_[:, :, None, :ns], v_[:, :, None, :ns]
    a = (qr @ kb.transpose(-1, -2) * scale).masked_fill(~near, -math.inf)
    b = (qr @ ks.transpose(-1, -2) * scale).masked_fill(~far, -math.inf)
    m = a.amax(-1, keepdim=True)
    m = torch.maximum(m, b.amax(-1, keepdim=True)) if ns else m
    m = torch.where(live, m, zero)
    a, b = (a - m).exp(), (b - m).exp()
    total = a.sum(-1, keepdim=True) + b.sum(-1, keepdim=True)
    inv = torch.where(live, 1.0 / total, zero)
    a, b = a * inv, b * inv
    o = a @ vb + b @ vs
    out = unrows(o).to(q.dtype)
    if not c["train"]:
        return out
    do = rows(torch.where(own_row, s["do"].float(), zero))
    delta = (do * o).sum(-1, keepdim=True)
    da, db = a * (do @ vb.transpose(-1, -2) - delta), b * (do @ vs.transpose(-1, -2) - delta)
    dq = (da @ kb + db @ ks) * scale
    dk = _unbanded(da.transpose(-1, -2) @ qr, N) * scale
    dv = _unbanded(a.transpose(-1, -2) @ do, N)
    dk[:, :, :ns] += (db.transpose(-1, -2) @ qr).sum(2) * scale
    dv[:, :, :ns] += (b.transpose(-1, -2) @ do).sum(2)
    return out, unrows(dq).to(q.dtype), dk.to(k.dtype), dv.to(v.dtype)


def _slots(s, at):
    """Page and place in it of position `at` [B, n] of each sequence."""
    page = s["k_cache"].shape[2]
    return s["page_table"].gather(1, torch.div(at, page, rounding_mode="floor")).long(), at % page


def _plain_append(s):
    q, k, v = s["q"], s["k"], s["v"]
    T = q.shape[2]
    new, first = s["new_lens"].long()[:, None], (s["lens"] - s["new_lens"]).long()[:, None]
    t = torch.arange(T, device=q.device)
    is_new = t < new
    page, place = _slots(s, torch.where(is_new, first + t, 0))
    page, place = page[is_new], place[is_new]
    s["k_cache"][page, :, place] = _rotate(k, s["pos"], s["tables"]).transpose(1, 2)[is_new]
    s["v_cache"][page, :, place] = v.transpose(1, 2)[is_new]
    return _rotate(q, s["pos"], s["tables"]), s["k_cache"], s["v_cache"]


def _plain_decode(s):
    c, q = s["case"], s["q"]
    B, Hq, _, d = q.shape
    Hkv, page = s["k_cache"].shape[1], s["k_cache"].shape[2]
    W, ns = min(c["window"], c["ctx"]), min(c["n_sink"], c["ctx"])
    length = s["lens"].long()[:, None]
    at = torch.cat([torch.arange(ns, device=q.device).expand(B, ns), length - W + torch.arange(W, device=q.device)], 1)
    first = torch.arange(ns + W, device=q.device) < ns
    see = torch.where(first, at < length - W, at >= 0)
    pg, place = _slots(s, torch.where(see, at, 0))
    k = s["k_cache"][pg, :, place].float().permute(0, 2, 1, 3)                 # [B, Hkv, ns + W, d]
    v = s["v_cache"][pg, :, place].float().permute(0, 2, 1, 3)
    v = torch.where(see[:, None, :, None], v, torch.zeros((), device=q.device))
    sc = (q.float().view(B, Hkv, Hq // Hkv, d) @ k.transpose(-1, -2) * s["sm_scale"]).masked_fill(~see[:, None, None], -math.inf)
    p = (sc - sc.amax(-1, keepdim=True)).exp()
    o = (p / p.sum(-1, keepdim=True)) @ v
    return o.view(B, Hq, 1, -1).to(q.dtype)


def run(state):
    s, c = state, state["case"]
    if own:
        import dl_templates_b200 as swa
        if c["op"] == "rope":
            q, k = s["q"], s["k"]
            if not c["train"]:
                return swa.RotaryPEAxes.apply(q, k, s["pos"], *s["tables"])
            q, k = q.detach().requires_grad_(), k.detach().requires_grad_()
            y = swa.RotaryPEAxes.apply(q, k, s["pos"], *s["tables"])
            return (*(t.detach() for t in y), *torch.autograd.grad(y, (q, k), (s["dq"], s["dk"])))
        if c["op"] == "attn":
            tail = (s["lens"], c["window"], c["n_sink"], s["sm_scale"])
            if not c["train"]:
                return swa.SinkSwa.apply(s["q"], s["k"], s["v"], *tail)
            x = [s[n].detach().requires_grad_() for n in ("q", "k", "v")]
            o = swa.SinkSwa.apply(*x, *tail)
            return (o.detach(), *torch.autograd.grad(o, x, s["do"]))
        if c["op"] == "append":
            q = swa.kv_append_rope(s["q"], s["k"], s["v"], s["pos"], s["tables"], s["k_cache"], s["v_cache"], s["page_table"],
                                   s["lens"], s["new_lens"])
            return q, s["k_cache"], s["v_cache"]
        return swa.sink_swa_decode(s["q"], s["k_cache"], s["v_cache"], s["page_table"], s["lens"], c["window"], c["n_sink"],
                                   s["sm_scale"])
    if c["op"] == "rope":
        y = _rotate(s["q"], s["pos"], s["tables"]), _rotate(s["k"], s["pos"], s["tables"])
        if c["train"]:
            y += _rotate(s["dq"], s["pos"], s["tables"], -1.0), _rotate(s["dk"], s["pos"], s["tables"], -1.0)
        return y
    return {"attn": _plain_attn, "append": _plain_append, "decode": _plain_decode}[c["op"]](s)


# ---- what a pass cannot do without -------------------------------------------------------------------------------------------
def _pairs(n, W, ns):
    """Query-key pairs of one head of a sequence of n tokens."""
    W = min(W, n)
    full = W * (W + 1) // 2 + (n - W) * W
    m = n - W                          # rows with something behind their window: row r of them has r + 1 tokens there
    s = min(ns, m)
    return full + s * (s + 1) // 2 + (m - s) * s


def _size(case):
    return 4 if case["dtype"] == "fp32" else 2


def _work_attn(c):
    e, B, Hq, Hkv = _size(c), c["B"], c["Hq"], c["Hkv"]
    lens = _lens(B, c["N"], c["ragged"])
    pairs = sum(_pairs(n, c["window"], c["n_sink"]) for n in lens) * Hq
    n_in, n_out = sum(lens), B * c["N"]
    qkv = n_in * (Hq * c["dqk"] + Hkv * (c["dqk"] + c["dv"]))
    flops = 2 * pairs * (c["dqk"] + c["dv"])
    nbytes = e * (qkv + n_out * Hq * c["dv"])
    if c["train"]:
        flops += 2 * pairs * (3 * c["dqk"] + 2 * c["dv"])
        nbytes += e * (n_in * Hq * c["dv"] + n_out * (Hq * c["dqk"] + Hkv * (c["dqk"] + c["dv"])))
    return {"bytes": nbytes, "flops": flops}


def work(case):
    c = case
    e, B, Hq, Hkv, dqk = _size(c), c["B"], c["Hq"], c["Hkv"], c["dqk"]
    if c["op"] == "attn":
        return _work_attn(c)
    pairs = c.get("r0", 0) + c.get("r1", 0) + c.get("r2", 0)
    axes = (c.get("r0", 0) > 0) + (c.get("r1", 0) > 0) + (c.get("r2", 0) > 0)
    if c["op"] == "rope":
        passes = 2 if c["train"] else 1
        return {"bytes": passes * B * c["N"] * (2 * e * (Hq + Hkv) * dqk + 4 * axes), "flops": passes * B * c["N"] * (Hq + Hkv) * 6 * pairs}
    lens = _lens(B, c["ctx"], c["ragged"])
    if c["op"] == "append":
        n = sum(min(a, b) for a, b in zip(_lens(B, c["N"], c["ragged"] and c["N"] > 1), lens))
        return {"bytes": 2 * e * (B * c["N"] * Hq * dqk + n * Hkv * (dqk + c["dv"])) + B * c["N"] * 4 * axes,
                "flops": (B * c["N"] * Hq + n * Hkv) * 6 * pairs}
    seen = sum(min(n, c["window"] + c["n_sink"]) for n in lens)
    return {"bytes": e * (seen * Hkv * (dqk + c["dv"]) + B * Hq * (dqk + c["dv"])), "flops": 2 * seen * Hq * (dqk + c["dv"])}


# ---- the definition in 64 bits, row by row of the mask -----------------------------------------------------------------------
def _exact_rotate(x, pos, tables, inverse=False):
    x = x.double()
    y = x.clone()
    at = 0
    for a, tab in enumerate(tables):
        R = tab.shape[1]
        z = torch.complex(tab[..., 0].double(), tab[..., 1].double())[pos[:, a].clamp(min=0).long()]
        z = torch.where((pos[:, a] < 0)[..., None], torch.ones_like(z), z)[:, None]
        w = torch.complex(x[..., at:at + R], x[..., at + R:at + 2 * R]) * (z.conj() if inverse else z)
        y[..., at:at + R], y[..., at + R:at + 2 * R] = w.real, w.imag
        at += 2 * R
    return y


def _exact_attn(s):
    c = s["case"]
    if c["Hq"] * c["B"] * c["N"] ** 2 > 6e9:
        return None
    q, k, v = (s[n].double() for n in ("q", "k", "v"))
    B, Hq, N, _ = q.shape
    G = Hq // k.shape[1]
    o = torch.zeros_like(s["q"][..., :1].expand(B, Hq, N, v.shape[-1]), dtype=torch.float64)
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    for b in range(B):
        n = N if s["lens"] is None else int(s["lens"][b])
        i = torch.arange(n, device=q.device)
        gap = i[:, None] - i[None, :]
        hidden = (gap < 0) | ((gap >= c["window"]) & (i[None, :] >= c["n_sink"]))
        for h in range(Hq):
            qh, kh, vh = q[b, h, :n], k[b, h // G, :n], v[b, h // G, :n]
            p = torch.softmax((qh @ kh.T * s["sm_scale"]).masked_fill_(hidden, -math.inf), -1)
            o[b, h, :n] = p @ vh
            if c["train"]:
                g = s["do"][b, h, :n].double()
                dv[b, h // G, :n] += p.T @ g
                ds = p * (g @ vh.T)
                ds -= p * ds.sum(-1, keepdim=True)
                dq[b, h, :n] = ds @ kh * s["sm_scale"]
                dk[b, h // G, :n] += ds.T @ qh * s["sm_scale"]
    return (o, dq, dk, dv) if c["train"] else o


def _exact_append(s):
    kc, vc = s["k_cache"].double(), s["v_cache"].double()
    page = kc.shape[2]
    k, v = _exact_rotate(s["k"], s["pos"], s["tables"]), s["v"].double()
    for b, (n, m) in enumerate(zip(s["lens"].tolist(), s["new_lens"].tolist())):
        at = torch.arange(n - m, n, device=kc.device)
        pages = s["page_table"][b][at // page].long()
        kc[pages, :, at % page] = k[b, :, :m].transpose(0, 1)
        vc[pages, :, at % page] = v[b, :, :m].transpose(0, 1)
    return _exact_rotate(s["q"], s["pos"], s["tables"]), kc, vc


def _exact_decode(s):
    c, page = s["case"], s["k_cache"].shape[2]
    out = []
    for b, n in enumerate(s["lens"].tolist()):
        at = torch.arange(n, device=s["q"].device)
        at = at[(at >= n - c["window"]) | (at < c["n_sink"])]
        pages = s["page_table"][b][at // page].long()
        k, v = (s[x][pages, :, at % page].double().transpose(0, 1) for x in ("k_cache", "v_cache"))
        q = s["q"][b, :, 0].double().unflatten(0, (k.shape[0], -1))
        out.append((torch.softmax(q @ k.mT * s["sm_scale"], -1) @ v).flatten(0, 1))
    return torch.stack(out)[:, :, None]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rope":
        y = _exact_rotate(s["q"], s["pos"], s["tables"]), _exact_rotate(s["k"], s["pos"], s["tables"])
        if case["train"]:
            y += _exact_rotate(s["dq"], s["pos"], s["tables"], True), _exact_rotate(s["dk"], s["pos"], s["tables"], True)
        return y
    return {"attn": _exact_attn, "append": _exact_append, "decode": _exact_decode}[case["op"]](s)
