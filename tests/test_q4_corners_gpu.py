"""The 4-bit operators (``q4``) where a mistake would hide: not-a-number and infinities in rows, weights and
queries, tensor scales at either end of fp32, readers whose exponent base moves again and again, cache rows that each
carry a mark of their own, and the sizes at which a variant begins.  The references are q4_reference's; the bounds are
counted as in test_q4_gpu.
"""
import numpy as np
import pytest
import torch

import q4_reference as ref
from conftest import pkg
from test_q4_gpu import CUDA, BF16, SCALE, U16, U32, History, bf, commit_setup, dev

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


# ------------------------------------------------------------------------------------ many steps a segment, marked rows
def base_moves(ctxs, scores, T, splits, W, H, sms):
    """How often the reader's exponent base moves after a segment's first step, restated: a CTA takes 128 rows a step;
    the base of a group of 8 heads starts at the first step's maxima and moves when a score passes its head's by 2^4.
    ``scores[t]``: log2 units, [H, n]."""
    cost = [2 * ((c - 1) // 128 + 1) + 1 if c > 0 else 0 for c in ctxs]
    need, per = T * splits * H * (W + 1), H * (W + 1)
    slots = (need - 2 * T) // per
    g = min(sms, slots - T + 1)
    segments = []
    if splits >= 2 and T <= 1024 and g >= 1:
        pref = np.concatenate(([0], np.cumsum(cost)))
        P = int(pref[-1])
        G = min(g, max(P // 2, 1))
        for cta in range(G):
            a, b = cta * P // G, (cta + 1) * P // G
            for t in range(T):
                lo, hi = max(a, pref[t]) - pref[t], min(b, pref[t + 1]) - pref[t]
                if lo >= hi:
                    continue
                step = lambda x: (x - 1) >> 1 if x > 0 else 0  # noqa: E731
                s0, s1 = step(lo), min(step(hi), (ctxs[t] + 127) // 128)
                if s0 < s1:
                    segments.append((t, s0, s1))
    else:
        segments = [(t, 0, (c + 127) // 128) for t, c in enumerate(ctxs) if c]
    moves = 0
    for t, s0, s1 in segments:
        for h0 in range(0, H, 8):
            s = scores[t][h0:h0 + 8]
            base = s[:, s0 * 128:s0 * 128 + 128].max(1)
            for i in range(s0 + 1, s1):
                x = s[:, i * 128:i * 128 + 128]
                if (x > base[:, None] + 4).any():
                    moves += 1
                    base = np.maximum(base, x.max(1))
    return moves, max((s1 - s0 for _, s0, s1 in segments), default=0)


class Marked(History):
    """Rows whose value half is zero but for one column, a mark of its own size; and keys that give a row the score the
    test wants: every key is the same pattern of signs, its scales rise (or not) with the row's position."""

    def __init__(self, ctxs, W, rise, heads, seed, H=16, page=16):
        super().__init__(ctxs, W=W, H=H, page=page, seed=seed, k_ts=2.0 ** -6, v_ts=0.5)
        rng = np.random.default_rng(seed)
        sign = rng.choice([-1, 1], W)
        flat = self.cache.reshape(-1).cpu().numpy().copy()
        kc, vc, ks, vs = ref.tile_views(flat, W)
        per = page // 16
        self.rows = []
        for t, n in enumerate(ctxs):
            if n == 0:
                self.rows.append((np.zeros((0, W)), np.zeros((0, W))))
                continue
            j = np.arange(n)
            tile, r = self.table[t, j // page].astype(np.int64) * per + (j % page) // 16, j % 16
            # scale bytes 56 (1.0) .. 96 (32.0) over the row's length: 8 levels a factor of two
            byte = np.full(n, 56) if rise == 0 else 56 + ((j if rise > 0 else n - 1 - j) * 41 // n)
            kn = np.broadcast_to(8 + 7 * sign, (n, W))
            kc[tile, :, r] = ref.words(kn).reshape(n, -1, 16)
            ks[tile, r] = byte[:, None]
            # value: column 61 j mod W, code 8 +- 1 .. 7, scale 2^-2 .. 2^1
            col = (61 * j + 7 * t) % W
            code = np.full((n, W), 8)
            code[j, col] = 8 + (1 + (j * 5 // W + j) % 7) * np.where((j // 3) % 2, 1, -1)
            vb = 40 + 8 * ((j * 3 + t) % 4)
            vc[tile, :, r] = ref.words(code).reshape(n, -1, 4)
            vs[tile, :, r] = vb[:, None]
            self.rows.append((7 * sign * ref.E4M3[byte][:, None] * self.k_ts, (code - 8) * ref.E4M3[vb][:, None] * self.v_ts))
        self.cache.copy_(dev(flat).view(self.cache.shape))
        # q . k = amp 7 k_ts s sum|sign| in the heads named, noise in the others
        amp = 2.0 * np.log(2) / (SCALE * 7 * self.k_ts * W)            # log2 units: 2 s, 2 .. 64
        self.q = bf(rng, len(ctxs), H, W, std=0.05)
        for h in heads:
            self.q[:, h] = ref.bf16(amp * (1 + (h % 3) / 4) * sign)
        self.qd = dev(self.q, BF16)

    def check(self, o, lse):
        """As History.check, with p's own rounding: 11 bits, half a step 2^-11 (f16), and no more."""
        o, lse = o.double().cpu().numpy(), lse.double().cpu().numpy()
        for t, (k, v) in enumerate(self.rows):
            eo, el, av, aq = ref.attention(self.q[t], k, v, SCALE)
            if k.shape[0] == 0:
                assert (o[t] == 0).all() and np.isneginf(lse[:, t]).all()
                continue
            d = (self.W / 16 + 8) * U32 * aq
            tol = ((2.0 ** -11 + 2 * d[:, None] + (k.shape[0] / 16 + 8) * U32) * av * 1.01 + U16 * 1.01 * np.abs(eo)
                   + 2.0 ** -36 * np.abs(v).sum(0))
            assert (np.abs(o[t] - eo) <= tol).all(), (t, (np.abs(o[t] - eo) / tol).max())
            assert (np.abs(lse[:, t] - el) <= d + 8 * U32 * (1 + np.abs(el)) + (k.shape[0] / 16 + 8) * U32).all(), t

    def log2_scores(self):
        return [self.q[t] @ k.T * SCALE / np.log(2) for t, (k, _) in enumerate(self.rows)]


@pytest.mark.parametrize('W', [256, 512, 1024])
@pytest.mark.parametrize('heads', [range(16), range(8), range(8, 16), (3,)])
def test_history_base_moves_many_times_in_a_segment(W, heads):
    """One CTA a row: 16 and 9 steps, the last ones short, the base moving in one group of heads or in both."""
    ctxs = [2047, 0, 1153, 130]
    h = Marked(ctxs, W, 1, heads, seed=W)
    moves, steps = base_moves(ctxs, h.log2_scores(), 4, 1, W, 16, 148)
    assert steps == 16 and moves >= 8 * (2 if len(heads) == 16 else 1), moves
    h.check(*h.run(splits=1))


@pytest.mark.parametrize('W,page', [(256, 32), (512, 16)])
def test_history_base_moves_in_a_batch_over_all_ctas(W, page):
    """70 rows of about 1000 over the whole GPU: CTAs take several steps and cross rows."""
    rng = np.random.default_rng(W)
    ctxs = rng.integers(700, 1300, 70).tolist() + [0, 5]
    h = Marked(ctxs, W, 1, range(16), seed=3, page=page)
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    moves, steps = base_moves(ctxs, h.log2_scores(), len(ctxs), 8, W, 16, sms)
    assert steps >= 4 and moves >= 60, (steps, moves)
    h.check(*h.run(splits=8))


@pytest.mark.parametrize('rise', [0, -1])
@pytest.mark.parametrize('ctxs,splits', [([5000], 64), ([5003, 129], 1), ([2100] * 9, 32), ([1029, 3], 64)])
@pytest.mark.parametrize('W', [256, 512])
def test_history_every_row_counts_once(W, ctxs, splits, rise):
    """Equal keys (each row's mark has the weight 1 / n) and falling ones: a row or tile that is left out, taken twice or
    put elsewhere is off by far more than the bound."""
    h = Marked(ctxs, W, rise, range(16), seed=len(ctxs) + W)
    h.check(*h.run(splits=splits))


@pytest.mark.parametrize('W,T,most', [(256, 1030, 140), (512, 1026, 40)])
def test_history_above_1024_rows(W, T, most):
    """One CTA a row, several rows a CTA, all heads, rows of more than one step."""
    rng = np.random.default_rng(T)
    ctxs = rng.integers(0, most, T).tolist()
    ctxs[7], ctxs[T - 1] = 300, 200
    h = History(ctxs, W=W, seed=4, poison=False)
    h.check(*h.run(splits=2))


# ------------------------------------------------------------------------------------ sizes at which a variant begins
@pytest.mark.parametrize('T,N,K', [(32, 10000, 64), (64, 9480, 128), (48, 10001, 2048), (33, 9473, 416)])
@pytest.mark.parametrize('residual', [False, True])
def test_linear_large_tiles_with_few_tokens(T, N, K, residual):
    from test_q4_gpu import test_linear
    test_linear(T, N, K, residual)


@pytest.mark.parametrize('T,N', [(3, 256), (20, 256), (40, 1200), (130, 256), (300, 2000), (1030, 2001)])
def test_linear_leaves_the_error_word_alone(T, N):
    """Every kernel with an error word: nothing in it after a call that went well, and the same output."""
    q4 = pkg('q4')
    rng = np.random.default_rng(T)
    w = q4.Weight.of(dev(bf(rng, N, 512), BF16))
    x = dev(bf(rng, T, 512), BF16)
    flag = torch.zeros(1, dtype=torch.int32, device=CUDA)
    assert torch.equal(w.linear(x, error_flag=flag), w.linear(x)) and flag.item() == 0


@pytest.mark.parametrize('share,W', [([18000, 1, 950], 512), ([37000, 0, 900, 7], 256)])
def test_commit_of_a_prompt_at_the_usual_widths(share, W):
    """Enough tokens for several rows a thread, at the widths of the two latents; rows nobody commits stay."""
    q4 = pkg('q4')
    c = commit_setup(share, W, 16, seed=W, padding=5)
    cache = torch.full((c['nb'], 1, 16, 17 * W // 16), 0x5a, dtype=torch.uint8, device=CUDA)
    slots = q4.commit_rows(dev(c['row'], BF16), dev(c['pos']), dev(c['table'], BF16), cache, dev(c['bt']), dev(c['qsl']),
                           0.25, 2.0)
    assert np.array_equal(slots.cpu().numpy(), c['slots'])
    real = c['slots'] >= 0
    rotated = ref.rope(c['row'][:, :W], c['table'], c['pos'])
    want = np.concatenate((ref.stored(rotated, 0.25), ref.stored(c['row'][:, W:], 2.0)), 1)
    got = q4.gather_slots(cache, slots, 0.25, 2.0).double().cpu().numpy()
    assert np.array_equal(got[real], want[real]) and (got[~real] == 0).all()
    free = np.setdiff1d(np.arange(c['nb'] * 16), c['slots'][real])
    for view, axis in zip(ref.tile_views(cache.cpu().numpy().reshape(-1), W), (2, 2, 1, 2)):
        assert (np.moveaxis(view, axis, 1).reshape(c['nb'] * 16, -1)[free] == 0x5a).all()


# ------------------------------------------------------------------------------------ partials into the sequence split
@pytest.mark.parametrize('width', [512, 256])
@pytest.mark.parametrize('parts', [1, 3])
def test_partials_go_into_the_exchange_and_the_combine(width, parts):
    """The slices of a sequence split over a 4-bit cache, one after the other on this GPU: partials, the reduce that
    stores exchange words, the combine that merges them, against the oracle over the values the cache stands for."""
    from test_attend_gpu import build_step, oracle
    from test_seqsplit_one_gpu import O_TOL, SplitStep
    lib = pkg('_lib')
    s = build_step(50 + parts, width, [3000, 40, 900, 0, 33, 31])
    lat = s['lat'].astype(np.float64)
    lat[0] = 0
    k_ts, v_ts = 2.0 ** -9, 2.0 ** -10
    nb = lat.shape[0]
    cache = np.zeros((nb, 1, 16, 17 * width // 16), dtype=np.uint8)
    views = ref.tile_views(cache.reshape(-1), width)
    kn, kb = ref.quantize(lat[:, 0, :, :width], k_ts)
    vn, vb = ref.quantize(lat[:, 0, :, width:], v_ts)
    views[0][:] = ref.words(kn).reshape(nb, 16, -1, 16).transpose(0, 2, 1, 3)
    views[1][:] = ref.words(vn).reshape(nb, 16, -1, 4).transpose(0, 2, 1, 3)
    views[2][:], views[3][:] = kb, vb.transpose(0, 2, 1)
    cache[0] = 0xff                                             # stale table columns name block 0
    s['lat'] = np.concatenate((ref.stored(lat[..., :width], k_ts), ref.stored(lat[..., width:], v_ts)), -1).astype(np.float32)
    kk, vv = ref.unpack_cache(cache[1:], width)
    assert np.array_equal(kk * k_ts, s['lat'][1:, 0, :, :width]) and np.array_equal(vv * v_ts, s['lat'][1:, 0, :, width:])

    class Split(SplitStep):
        def reduce_slice(self, r, world=None):
            table, rows = self.slices[r]
            stream = lib.stream_of(self.q_lat)
            lib.call('hla_s6_history_partials_q4', lib.ptr(self.q_lat), self.q_lat.stride(0), self.q_lat.stride(1),
                     lib.ptr(self.four), nb, self.four.stride(0), lib.ptr(table), table.stride(0), table.shape[1],
                     lib.ptr(rows), self.T, 16, self.W, 16, float(self.scale), self.splits, lib.ptr(self.ws),
                     self.ws_floats, k_ts, v_ts, lib.ptr(self.err), 0, stream)
            parts = [self.recv[d, r].data_ptr() for d in range(self.D)]
            lib.call('hla_s6_history_reduce_exchange', self.T, 16, self.W, 16, self.splits, lib.ptr(self.ws),
                     self.ws_floats, None, lib.pointer_array(parts), lib.ptr(self.epochs), self.D, 0, stream)

    run = Split(s, parts, parts)
    run.four = dev(cache)
    want = oracle(s, run.scale)
    for step in range(2):
        for out in run.step():
            got = out.float().cpu().numpy()
            assert (got[s['R']:] == 0).all()
            np.testing.assert_allclose(got, want, **O_TOL)
    assert int(run.err.item()) == 0 and (run.epochs == 2).all()


def test_commit_with_more_requests_than_fit_shared_memory():
    """1100 requests of one token, some padding: the kernel searches the request list in global memory."""
    q4 = pkg('q4')
    W = 256
    c = commit_setup([1, 0, 2] * 367, W, 16, seed=6, padding=3, start=[i % 50 for i in range(1101)])
    cache = q4.new_cache(c['nb'], 16, W)
    slots = q4.commit_rows(dev(c['row'], BF16), dev(c['pos']), dev(c['table'], BF16), cache, dev(c['bt']), dev(c['qsl']))
    assert np.array_equal(slots.cpu().numpy(), c['slots'])
    real = c['slots'] >= 0
    rotated = ref.rope(c['row'][:, :W], c['table'], c['pos'])
    want = np.concatenate((ref.stored(rotated, 1.0), ref.stored(c['row'][:, W:], 1.0)), 1)
    assert np.array_equal(q4.gather_slots(cache, slots).double().cpu().numpy()[real], want[real])
