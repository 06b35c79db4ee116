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
