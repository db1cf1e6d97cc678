"""The 4-bit operators (``q4``) where a mistake would hide: not-a-number and infinities in rows, weights and
queries, and tensor scales at either end of fp32.  The references are q4_reference's; the bounds are counted as in
test_q4_gpu.
"""
import numpy as np
import pytest
import torch

import q4_reference as ref
from conftest import pkg
from test_q4_gpu import CUDA, BF16, History, bf, commit_setup, dev

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


# ------------------------------------------------------------------------------------ the reader and values not finite
def check_but(h, o, lse, touched):
    """``History.check`` with the (token, head) pairs of ``touched`` taken from a run with the queries ``h.q``."""
    clean_o, clean_lse = h.run(q=dev(h.q, BF16))
    for t, hd in touched:
        o[t, hd], lse[hd, t] = clean_o[t, hd], clean_lse[hd, t]
    h.check(o, lse)


@pytest.mark.parametrize('ctxs,splits', [([40], 64), ([5000], 64), ([900, 0, 17], 1), ([300] * 20 + [0, 1], 16)])
@pytest.mark.parametrize('W', [256, 512])
def test_history_nan_in_a_query_stays_in_its_head(W, ctxs, splits):
    """A NaN query is a NaN row, one partial or many; rows without history are empty all the same."""
    h = History(ctxs, W=W, seed=7)
    touched = [(t, hd) for t, hd in ((0, 3), (0, 12), (len(ctxs) - 1, 0), (1, 5)) if t < len(ctxs)]
    for t, hd in touched:
        h.qd[t, hd, 9 * hd] = float('nan')
    o, lse = h.run(splits=splits)
    for t, hd in touched:
        if ctxs[t]:
            assert torch.isnan(o[t, hd]).all() and torch.isnan(lse[hd, t]), (t, hd)
        else:
            assert (o[t, hd] == 0).all() and torch.isneginf(lse[hd, t])
    check_but(h, o, lse, touched)


@pytest.mark.parametrize('splits', [1, 64])
def test_history_infinite_queries(splits):
    """Scores of +inf make a NaN row, as in exp(s - max) of the formula; a row whose scores are all -inf is empty."""
    ctxs = [200, 1500, 70]
    h = History(ctxs, W=256, seed=3)
    flat = h.cache.reshape(-1).cpu().numpy().copy()
    codes = ref.tile_views(flat, 256)[0][:, 0, :, 0]
    codes[:] = (codes & 0xf0) | 3                                # column 0 of every key: code 3, below zero
    h.cache.copy_(dev(flat).view(h.cache.shape))
    k, _ = ref.unpack_cache(h.cache.cpu().numpy(), 256)
    for t, n in enumerate(ctxs):
        rows = k[h.table[t, :-(-n // 16)]].reshape(-1, 256)[:n] * h.k_ts
        assert (rows[:, 0] < 0).all()
        h.rows[t] = (rows, h.rows[t][1])
    touched = [(0, 2), (1, 9), (1, 0), (2, 15)]
    for (t, hd), v in zip(touched, (np.inf, np.inf, -np.inf, -np.inf)):
        h.qd[t, hd, 0] = v
    o, lse = h.run(splits=splits)
    for t, hd in ((0, 2), (1, 9)):
        assert (o[t, hd] == 0).all() and torch.isneginf(lse[hd, t]), (t, hd)
    for t, hd in ((1, 0), (2, 15)):
        assert torch.isnan(o[t, hd]).all() and torch.isnan(lse[hd, t]), (t, hd)
    check_but(h, o, lse, touched)


@pytest.mark.parametrize('ctxs,splits', [([40, 64], 64), ([3000, 500], 64), ([700, 130], 1)])
def test_history_nan_in_a_cached_row_stays_in_its_request(ctxs, splits):
    """A NaN key makes its request's rows NaN in every head, a NaN group of a value row that group's columns."""
    W = 512
    h = History(ctxs, W=W, seed=2)
    clean = h.run(splits=splits)
    at = ctxs[0] // 2
    flat = h.cache.reshape(-1).cpu().numpy().copy()
    views = ref.tile_views(flat, W)
    tile, r = h.table[0, at // 16], at % 16
    old = views[3][tile, 4, r]
    views[3][tile, 4, r] = 0x7f                                 # V columns 128 .. 159
    h.cache.copy_(dev(flat).view(h.cache.shape))
    o, lse = h.run(splits=splits)
    assert torch.isnan(o[0, :, 128:160]).all() and torch.equal(lse, clean[1])
    keep = torch.tensor([c for c in range(W) if not 128 <= c < 160], device=CUDA)
    assert torch.equal(o[0][:, keep], clean[0][0][:, keep]) and torch.equal(o[1], clean[0][1])
    views[3][tile, 4, r] = old
    views[2][tile, r, 15] = 0x7f                                # K columns 480 .. 511
    h.cache.copy_(dev(flat).view(h.cache.shape))
    o, lse = h.run(splits=splits)
    assert torch.isnan(o[0]).all() and torch.isnan(lse[:, 0]).all()
    assert torch.equal(o[1], clean[0][1]) and torch.equal(lse[:, 1], clean[1][:, 1])


def test_attend_keeps_a_nan_query_in_its_head():
    """Through the fused combine: NaN in that head of that token, every other output bit as before."""
    from test_q4_chain_gpu import Layer
    lay = pkg('s6_layer')
    layer = Layer(16, 256, 512, 256, 32, 16, seed=21)
    layer.run([(0, 60), (1, 100)])
    ctx, *_ = layer.step([(0, 1), (1, 1)])
    T, H, loop = 2, 16, 1
    q, v = layer.rnd(T, H, 128), layer.rnd(T, H, 128)
    exact = torch.nan_to_num(layer.caches.exact[loop]).transpose(1, 2)
    q_lat = layer.rnd(T, H, 512, std=0.5)
    call = lambda: lay.attend(layer.sl, loop, q_lat, q, None, v, layer.caches.main, layer.caches.latent_table,  # noqa: E731
                              *layer.caches.main_scale, ctx, (exact, layer.caches.exact_table))
    was = call()
    assert torch.isfinite(was).all()
    q_lat[1, 6, 100] = float('nan')
    got = call()
    assert torch.isnan(got[1, 6]).all()
    got[1, 6] = was[1, 6]
    assert torch.equal(got, was)


# ------------------------------------------------------------------------------------ tensor scales at either end
@pytest.mark.parametrize('ts', [2.0 ** -126, 2.0 ** -124, 2.0 ** -119, 2.0 ** -118, 2.0 ** -117, 2.0 ** -100, 2.0 ** 100,
                                2.0 ** 115, 2.0 ** 116, 2.0 ** 117, 2.0 ** 120, 2.0 ** 123, 2.0 ** 126, 2.0 ** 127,
                                1.5 * 2.0 ** -125, 1.5 * 2.0 ** 126])
def test_commit_at_the_ends_of_the_tensor_scales(ts):
    """Codes and scales are the formula's for every tensor scale, infinities included.  (1.5: exact as 3 / 8 is.)"""
    q4 = pkg('q4')
    W = 256
    c = commit_setup([24], W, 16, seed=1)
    rng = np.random.default_rng(int(np.log2(ts)) & 255)
    spread = np.exp2(rng.integers(-14, 13, (24, 2 * W // 32))).repeat(32, 1)
    with np.errstate(over='ignore'):
        x = torch.from_numpy(np.clip(rng.standard_normal((24, 2 * W)) * spread * ts, -3e38, 3e38)).to(BF16).double().numpy()
    assert np.isfinite(x).all()
    x[3, W:] = 0
    x[5, W + 3], x[5, W + 4] = np.inf, -np.inf
    x[6, :W // 2] = 0
    x[6, 1] = -np.inf
    c['table'][:, :W // 2], c['table'][:, W // 2:] = 1, 0       # the identity rotation
    x[:, W // 2:W] = 0                                          # (inf * 0 of a partner would be NaN)
    key = x[:, :W].copy()
    key[6, W // 2 + 1] = np.nan
    want = np.zeros((c['nb'], 1, 16, 17 * W // 16), dtype=np.uint8)
    for t, s in enumerate(c['slots']):
        ref.put_row(want, W, 16, int(s), np.nan_to_num(key[t], nan=0.0, posinf=np.inf, neginf=-np.inf), x[t, W:], ts, ts)
    cache = dev(np.zeros_like(want))
    q4.commit_rows(dev(x, BF16), dev(c['pos']), dev(c['table'], BF16), cache, dev(c['bt']), dev(c['qsl']), ts, ts)
    got = cache.cpu().numpy()
    slot = int(c['slots'][6])                                   # the partner's group holds a NaN: not compared here
    for a in (got, want):
        views = ref.tile_views(a[slot // 16].reshape(-1), W)
        views[0][:, (W // 2 + 1) // 32, slot % 16] = 0
        views[2][:, slot % 16, (W // 2 + 1) // 32] = 0
    np.testing.assert_array_equal(got, want)
    if 2.0 ** -110 < ts < 2.0 ** 110:                           # (beyond, values leave bf16's range)
        back = q4.gather_slots(dev(want), dev(c['slots']), ts, ts).double().cpu().numpy()
        np.testing.assert_array_equal(back[:, W:], ref.stored(x[:, W:], ts))


@pytest.mark.parametrize('amax', [1e-38, 3e-36, 3.3e38])
def test_weights_of_tiny_and_huge_values(amax):
    """``quantize_weight`` picks its scale: the packed values are the formula's and within half a step of the weight."""
    q4 = pkg('q4')
    rng = np.random.default_rng(0)
    w = torch.from_numpy(rng.uniform(-amax, amax, (48, 160))).to(BF16)
    packed, scale = q4.quantize_weight(w.to(CUDA))
    n, b = ref.quantize(w.double().numpy(), scale)
    got = ref.unpack_weight(packed.cpu().numpy(), 48, 160)
    np.testing.assert_array_equal(got, (n - 8) * np.repeat(ref.E4M3[b], 32, -1))
    err = np.abs(got * scale - w.double().numpy()).reshape(48, -1, 32)
    assert (err <= np.abs(w.double().numpy()).reshape(48, -1, 32).max(-1, keepdims=True) / 7 * (1 + 2.0 ** -4) / 2).all()
