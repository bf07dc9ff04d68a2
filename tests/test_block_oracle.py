"""CPU: the residual-block oracle (oracle/block_oracle.py) against published vectors and simple
restatements, and the refusals of the block entry points (their checks come before any device
call, so they run without a GPU)."""
import ctypes

import numpy as np
import pytest

import block_oracle as BO
import dcn_runtime as rt

OK_PTR = 1 << 20  # an aligned non-null address; refused calls never read it


@pytest.mark.parametrize("ctr,key,want", [
    # the published known answers of philox4x32 with 10 rounds
    ((0, 0, 0, 0), (0, 0), (0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8)),
    ((BO.M32,) * 4, (BO.M32,) * 2, (0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd)),
    ((0x243f6a88, 0x85a308d3, 0x13198a2e, 0x03707344), (0xa4093822, 0x299f31d0),
     (0xd16cfe09, 0x94fdcceb, 0x5001e420, 0x24126ea1)),
])
def test_philox_known_answers(ctr, key, want):
    assert tuple(BO.philox4x32_10(ctr, key)) == want


@pytest.mark.parametrize("first", [0, 5, 8 * 2**32 - 3])
def test_draws_follow_the_scalar_generator(first):
    seed, off = 0x123456789ABCDEF0, 0xFEDCBA9876543210
    got = BO.draws(first, 21, seed, off)
    for j, u in enumerate(got):
        i = first + j
        w = BO.philox4x32_10(((i >> 3) & BO.M32, i >> 35, off & BO.M32, off >> 32),
                             (seed & BO.M32, seed >> 32))
        assert u == (w[(i & 7) >> 1] >> (16 * (i & 1))) & 0xFFFF


def _dropout(L, res=None, y=OK_PTR * 2, x=OK_PTR, rng=None, **kw):
    d = rt.DropoutDesc(**{**dict(n=64, group=1, dtype=rt.DCN_F32, p=0.5), **kw})
    return L.dcn_dropout_fwd(None, ctypes.byref(d), x, res, y, rng)


@pytest.mark.parametrize("kw,msg", [
    (dict(p=-0.1), "0 <= p <= 1"), (dict(p=1.5), "0 <= p <= 1"), (dict(p=float("nan")), "p <= 1"),
    (dict(n=-1), "element count"), (dict(group=0), "group"), (dict(dtype=2), "dtype"),
    (dict(x=None), "null tensor"), (dict(y=None), "null tensor"),
    (dict(x=OK_PTR + 2), "aligned"), (dict(rng=OK_PTR * 8 + 4), "8-byte"),
    (dict(y=OK_PTR + 16), "overlaps"), (dict(res=OK_PTR * 2 + 4), "overlaps"),
    (dict(rng=OK_PTR * 2 + 8), "overlaps"),
    (dict(), "null handle"),  # everything right but the handle
    (dict(y=OK_PTR), "null handle"), (dict(res=OK_PTR * 2), "null handle"),  # in place
])
def test_dropout_refusals(kw, msg):
    L = rt.load()
    assert _dropout(L, **kw) == -1
    assert msg in rt.last_error()


def test_null_descriptor():
    L = rt.load()
    assert L.dcn_dropout_fwd(None, None, OK_PTR, None, OK_PTR * 2, None) == -1


def test_drop_factor_mean():
    """The kept share of 2^20 draws is within 5 standard deviations of 1 - p, and the factor's
    mean within the same of 1."""
    n, p = 1 << 20, 0.1
    f = BO.drop_factor(n, 1, p, 7, 3)
    sd = (p * (1 - p) / n) ** 0.5
    assert abs(np.mean(f > 0) - (1 - p)) < 5 * sd + 1 / 65536
    assert abs(f.mean() - 1) < 5 * sd / (1 - p)
