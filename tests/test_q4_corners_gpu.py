"""The 4-bit operators (``q4``) where a mistake would hide: not-a-number and infinities in rows and weights.  The
references are q4_reference's.
"""
import numpy as np
import pytest
import torch

import q4_reference as ref
from conftest import pkg
from test_q4_gpu import BF16, bf, commit_setup, dev

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------ rows and weights with a NaN
def nan_groups(x, ts):
    """The values ``x`` (may hold NaN) is stored as: a group with a NaN reads back as NaN throughout."""
    bad = np.isnan(x.reshape(*x.shape[:-1], -1, 32)).any(-1)
    out = ref.stored(np.where(np.isnan(x), 0.0, x), ts)
    out[np.repeat(bad, 32, -1)] = np.nan
    return out


@pytest.mark.parametrize('W', [256, 512, 1024])
@pytest.mark.parametrize('k_ts,v_ts', [(0.25, 2.0), (0.375, 5.0)])
def test_a_nan_in_a_committed_row_is_kept(W, k_ts, v_ts):
    q4 = pkg('q4')
    c = commit_setup([7], W, 16, seed=W)
    row = c['row'].copy()
    row[1, W + 5] = np.nan                                      # V alone
    row[2, 7] = np.nan                                          # K: its rotation partner W / 2 further too
    row[3, W + 33], row[3, W + 34] = np.nan, np.inf             # beside an infinity
    row[4, W:] = np.nan
    row[5, 2 * W - 1] = -np.nan
    c['table'][:, :W // 2], c['table'][:, W // 2:] = 1, 0       # the identity rotation
    cache = q4.new_cache(c['nb'], 16, W)
    slots = q4.commit_rows(dev(row, BF16), dev(c['pos']), dev(c['table'], BF16), cache, dev(c['bt']), dev(c['qsl']),
                           k_ts, v_ts)
    got = q4.gather_slots(cache, slots, k_ts, v_ts).double().cpu().numpy()
    key = row[:, :W].copy()
    key[2, 7 + W // 2] = np.nan                                 # NaN * 0 enters its partner
    for half, x, ts in ((got[:, :W], key, k_ts), (got[:, W:], row[:, W:], v_ts)):
        # (a value (n - 8) s ts with ts = 3 / 8 or 5 has up to 9 bits: the gather rounds it to bf16)
        np.testing.assert_array_equal(half, ref.bf16(nan_groups(x, ts)))
    scales = ref.tile_views(cache[slots[4] // 16].cpu().numpy().reshape(-1), W)[3]
    assert (scales[0, :, slots[4].item() % 16] == 0x7f).all()


@pytest.mark.parametrize('T', [1, 40, 200, 1030])
def test_a_nan_in_a_weight_is_kept(T):
    """Packed with a given scale (without one ``quantize_weight`` refuses it): its output is NaN, the others are not."""
    q4 = pkg('q4')
    N, K = 2001, 256
    rng = np.random.default_rng(T)
    w, x = bf(rng, N, K, std=K ** -0.5), bf(rng, T, K)
    w[1999, 70] = np.nan
    with pytest.raises(ValueError, match='not finite'):
        q4.quantize_weight(dev(w, BF16))
    packed, scale = q4.quantize_weight(dev(w, BF16), 0.0078125)
    y = q4.linear(dev(x, BF16), packed, N, scale)
    assert torch.isnan(y[:, 1999]).all()
    keep = [n for n in range(N) if n != 1999]
    assert torch.isfinite(y[:, keep]).all()
    clean, _ = q4.quantize_weight(dev(np.nan_to_num(w), BF16), 0.0078125)
    assert torch.equal(y[:, keep], q4.linear(dev(x, BF16), clean, N, scale)[:, keep])
