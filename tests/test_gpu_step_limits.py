"""The step operators at the ends of their ranges.

Tolerances count roundings, u = 2^-24.  A norm's sum of squares: a thread adds the values of the vectors that it holds one
after another (at most 64), and what it reads beyond them a vector at a time, compensated (8 additions and 2); then 5
exchanges of a warp, at most 8 warps, one value behind the last whole vector.  So 80 u of the sum for any length, 40 u of
its root; 6 more for the mean, eps, root, reciprocal and products; and the output's own rounding.
"""
import math

import numpy as np
import pytest
import torch

from test_gpu_step import INF, KINDS, U, normal

pytestmark = pytest.mark.gpu

u = 2.0 ** -24
NORM = 46 * u


@pytest.fixture(scope="module")
def S(dev):
    from vdttfs import seq
    return seq


# ------------------------------------------------------- norms of long rows --
def check_long(S, x, residual=None, weight=None):
    total = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    z = total.float() if weight is None else total.float() * weight.float()
    root = (total.double().square().mean(1, keepdim=True) + 1e-6).sqrt()
    y, s = S.add_rms_norm(x, residual, weight)
    assert torch.equal(s, total)
    want = z.double() / root
    assert ((y.double() - want).abs() <= (U[x.dtype] + NORM) * want.abs() + (2.0 ** -25 if x.dtype == torch.float16 else 1e-37)).all()
    codes, scale, _ = S.add_rms_norm_int8(x, residual, weight)
    unit = z.abs().amax(1) * torch.tensor(np.float32(1) / np.float32(127)).cuda()
    want = unit.double() / root[:, 0]
    assert ((scale.double() - want).abs() <= NORM * want).all(), ((scale.double() / want - 1).abs().max() / u).item()
    assert torch.equal(codes.float(), torch.round(z / unit[:, None]))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("cols", [16391, 1 << 20, (1 << 22) + 5])
def test_norm_of_long_rows(S, kind, cols):
    """Rows of one value, whose squares round the same way at every addition, and random ones; on 16 bytes and off them."""
    x = torch.stack([torch.full((cols + 1,), 1.1), torch.full((cols + 1,), 0.37), normal(cols, cols + 1)]).to(kind).cuda()
    check_long(S, x[:, :cols])
    check_long(S, x[:, 1:])
    check_long(S, x[:, :cols], x[:, 1:].flip(0), (1 + 0.3 * normal(1, cols)).to(kind).cuda())


def test_norm_of_a_row_of_16_million(S):
    check_long(S, torch.full((1, 1 << 24), 1.7, device="cuda"))


def test_norm_of_long_rows_that_pass_32_bits(S):
    """The squares' sum past 3.4e38 gives a factor of 0, wherever in the row it passes; an infinity or a NaN in what is
    read beyond the held vectors is seen."""
    x = torch.ones(5, 70000, device="cuda")
    x[0, :4] = 1.5e19
    x[1, 60000:60004] = 1.5e19
    x[2, 69999] = INF
    x[3, 65000] = math.nan
    y, _ = S.add_rms_norm(x)
    codes, scale, _ = S.add_rms_norm_int8(x)
    assert (y[:2] == 0).all() and (scale[:2] == 0).all()
    assert (y[2, :-1] == 0).all() and torch.isnan(y[2, -1]) and torch.isnan(y[3]).all() and not torch.isfinite(scale[2:4]).any()
    assert ((y[4].double() - 1 / math.sqrt(1 + 1e-6)).abs() <= NORM + u).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("cols", [1000, 16384, 16391, 40003])
def test_norm_in_place_at_every_length(S, kind, cols):
    """Outputs over inputs, in rows that registers hold and in longer ones, which are read again."""
    x, r, w = normal(1, 5, cols, kind=kind).cuda(), normal(2, 5, cols, kind=kind).cuda(), (1 + 0.2 * normal(3, cols)).to(kind).cuda()
    y, t = S.add_rms_norm(x, r, w)
    codes, scale, _ = S.add_rms_norm_int8(x, r, w)
    alone = S.add_rms_norm(x, None, w)[0]
    for out, total in (("x", "r"), ("r", "x"), ("x", None), (None, "r"), (None, "x"), ("r", None)):
        a, b = x.clone(), r.clone()
        at = {"x": a, "r": b, None: None}
        got, s = S.add_rms_norm(a, b, w, out=at[out], sum_out=at[total])
        assert torch.equal(got, y) and torch.equal(s, t), (out, total)
        if out is None:
            a, b = x.clone(), r.clone()
            at = {"x": a, "r": b}
            for p, q in zip(S.add_rms_norm_int8(a, b, w, sum_out=at[total]), (codes, scale, t)):
                assert torch.equal(p, q), total
    a = x.clone()
    assert torch.equal(S.add_rms_norm(a, None, w, out=a)[0], alone)
    a = x.clone()
    assert torch.equal(S.add_rms_norm(a, a, w, sum_out=a)[0], S.add_rms_norm(x, x, w)[0])
