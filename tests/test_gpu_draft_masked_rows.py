"""Tree attention's rows without a finite score: the softmax over scores that are
all -Inf is NaN, as its formula has it, while a place without a token and a
sequence whose length does not fit give zeros.  In every form the kernels take:
unsplit, split and joined, few rows and many."""
from __future__ import annotations

import numpy as np
import pytest

import draft_ref as ref
from test_gpu_draft import val
from test_gpu_draft_numerics import FORMS, inputs, run

pytestmark = pytest.mark.gpu

NEG_INF, INF = 0xFF80, 0x7F80


def nans(wx, q, k, v, par, past, scale):
    """Where the formula in 64 bits is NaN, [B, t, heads, dh]."""
    with np.errstate(invalid="ignore"):
        return np.stack([np.isnan(ref.tree_attn(val(wx, q[b]), val(wx, k[b]), val(wx, v[b]), par[b], int(past[b]), scale)[0])
                         for b in range(len(past))])


def check(wx, be, q, k, v, par, past, clean=None):
    got, want = run(wx, be, q, k, v, par, past), nans(wx, q, k, v, par, past, q.shape[3] ** -0.5)
    np.testing.assert_array_equal(np.isnan(got), want)
    return got, want


@pytest.mark.parametrize("t,heads,kv,dh,past", FORMS)
def test_rows_of_no_finite_score_are_nan(wx, be, rng, t, heads, kv, dh, past):
    """Every key of one key head of sequence 0 is -Inf against positive queries."""
    print(f"all -inf t {t} heads {heads}/{kv} dh {dh} past {past}", flush=True)
    q, k, v, par, past = inputs(wx, rng, t, heads, kv, dh, past, positive=True)
    clean = run(wx, be, q, k, v, par, past)
    k[0, kv - 1] = NEG_INF
    got, want = check(wx, be, q, k, v, par, past)
    assert want[0, :, heads - heads // kv:].all() and want.sum() == t * (heads // kv) * dh
    np.testing.assert_array_equal(got[~want], clean[~want])


@pytest.mark.parametrize("t,heads,kv,dh", [(5, 4, 2, 64), (33, 4, 1, 128), (40, 8, 2, 128), (20, 3, 3, 256), (70, 2, 1, 256)])
def test_a_root_without_a_finite_score(wx, be, rng, t, heads, kv, dh):
    """Nothing cached; the roots' keys are -Inf: NaN for them, not for their children."""
    print(f"roots t {t} heads {heads}/{kv} dh {dh}", flush=True)
    q, k, v, par, past = inputs(wx, rng, t, heads, kv, dh, [0, 0], positive=True)
    par[0] = [-1 if i % 3 == 0 else i - i % 3 for i in range(t)]
    k[0, :, 0:t:3] = NEG_INF
    _, want = check(wx, be, q, k, v, par, past)
    assert (want[0].all((1, 2)) == (np.arange(t) % 3 == 0)).all()


@pytest.mark.parametrize("t,heads,kv,dh,past", FORMS)
def test_no_token_and_no_room_stay_zero(wx, be, rng, t, heads, kv, dh, past):
    """Places without a token, and sequences whose length does not fit, over -Inf keys."""
    print(f"zeros t {t} heads {heads}/{kv} dh {dh} past {past}", flush=True)
    q, k, v, par, past = inputs(wx, rng, t, heads, kv, dh, past, positive=True)
    k[:] = NEG_INF
    par[0, -1] = t + 7
    past[1] = -3
    got, _ = check(wx, be, q, k, v, par, past)
    assert not got[0, -1].any() and not got[1].any()
    past[1] = k.shape[2] - t + 1
    got, _ = check(wx, be, q, k, v, par, past)
    assert not got[0, -1].any() and not got[1].any()


@pytest.mark.parametrize("t,heads,kv,dh,past", FORMS)
def test_an_infinite_value_without_weight_is_nan(wx, be, rng, t, heads, kv, dh, past):
    """0 * Inf, the same wherever the slots' parts end: a whole run of cached keys
    of -Inf, as long as the parts of a split cache, with one Inf among their values."""
    print(f"0 inf t {t} heads {heads}/{kv} dh {dh} past {past}", flush=True)
    q, k, v, par, past = inputs(wx, rng, t, heads, kv, dh, past, positive=True)
    n = max(1, int(past[0]) - 70)
    k[0, :, :n] = NEG_INF
    v[0, 0, 9, n // 2] = INF
    got, want = check(wx, be, q, k, v, par, past)
    assert want[0, :, :heads // kv, 9].all() and want.sum() == t * (heads // kv)
