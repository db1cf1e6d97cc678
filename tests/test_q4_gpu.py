"""The 4-bit operators on the GPU (``q4``), against the format and formulas restated in float64 (q4_reference).

Error bounds, each a sum of roundings counted at half a step (bf16 2^-8, fp32 2^-24):

* commit and gather are exact: same codes, same scales, values exact in bf16 for power-of-two tensor scales.
* history: a score is an fp32 sum of exact products; a tensor-core step adds 16 products and truncates, so it is
  off by at most (W / 16 + 8) * 2^-22 * sum|q k| * scale =: d, which moves every p by a factor exp(+-2 d).  p is
  rounded for the value product (at most 2^-8 of sum p|v| / l); the sums over rows add (rows / 16 + 8) * 2^-22;
  the result is rounded once (2^-8 |o|).  lse is off by d plus a few fp32 steps.
  Small p: the kernel holds 2^11 p in f16, whose numbers below 2^-14 are multiples of 2^-24, so a p is off by at
  most 2^-25 / 2^11 = 2^-36 where that is more than its relative rounding (a p of e^-59 becomes 0).  p is relative
  to a base that is the maximum of some step's keys, so one key has p = 1 or more, l >= 1, and the error this adds
  to sum p v / l is at most 2^-36 sum|v|.
* linear: (K / 16 + 8) * 2^-22 * sum|x w| * scale, and the final rounding.
"""
import numpy as np
import pytest
import torch

import q4_reference as ref
from conftest import pkg

pytestmark = pytest.mark.gpu
CUDA, BF16 = 'cuda', torch.bfloat16
SCALE = 128 ** -0.5
U16, U32 = 2.0 ** -8, 2.0 ** -22


def dev(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a)).to(CUDA)
    return t.to(dtype) if dtype else t


def bf(rng, *shape, std=1.0):
    return ref.bf16(rng.standard_normal(shape) * std)


# ------------------------------------------------------------------------------------ history
class History:
    """A paged 4-bit cache with shuffled blocks, and each request's K and V rows as the reference sees them."""

    def __init__(self, ctxs, W=512, H=16, page=16, seed=0, k_ts=0.125, v_ts=0.25, pad=0, poison=True):
        rng = np.random.default_rng(seed)
        self.ctxs, self.W, self.H, self.page, self.k_ts, self.v_ts = list(ctxs), W, H, page, k_ts, v_ts
        T = len(self.ctxs)
        pages = [-(-c // page) for c in self.ctxs]
        nb = sum(pages) + 2
        cache, k, v = ref.random_cache(rng, nb, page, W)
        perm = rng.permutation(nb - 2) + 1
        width = max(pages + [1]) + 1
        self.table = rng.integers(0, nb, (T, width)).astype(np.int32)       # stale columns name live blocks
        used = np.zeros((nb, page), dtype=bool)
        self.rows, at = [], 0
        for t, n in enumerate(pages):
            blocks = perm[at:at + n]
            at += n
            self.table[t, :n] = blocks
            self.table[t, n:] = nb - 1                                      # block nb - 1 is poison
            used[blocks] = True
            if n:
                used[blocks[-1], (self.ctxs[t] - 1) % page + 1:] = False
            self.rows.append((k[blocks].reshape(-1, W)[:self.ctxs[t]] * k_ts,
                              v[blocks].reshape(-1, W)[:self.ctxs[t]] * v_ts))
        if poison:      # every byte of a row that no request owns is 0xff: codes 15, scales NaN
            views = ref.tile_views(cache.reshape(-1), W)
            dead = ~used.reshape(-1, 16)
            for i, r in np.argwhere(dead):
                views[0][i, :, r] = 255
                views[1][i, :, r] = 255
                views[2][i, r] = 255
                views[3][i, :, r] = 255
        self.q = bf(rng, T, H, W, std=0.5)
        full = torch.zeros(nb, page * 17 * W // 16 + pad, dtype=torch.uint8, device=CUDA)
        full[:, :page * 17 * W // 16] = dev(cache.reshape(nb, -1))
        self.cache = full.as_strided((nb, 1, page, 17 * W // 16), (full.stride(0), page * 17 * W // 16, 17 * W // 16, 1))
        self.bt, self.ctx = dev(self.table), dev(np.array(self.ctxs, dtype=np.int32))
        self.qd = dev(self.q, BF16)

    def run(self, splits=8, q=None, empty=None, ws=None, error_flag=None):
        ops, q4 = pkg('s6_ops'), pkg('q4')
        T = len(self.ctxs)
        ws = ws or ops.S6Workspace(self.H, self.W, max(T, 1) * splits)
        return q4.history_attention(self.qd if q is None else q, self.cache, self.bt, self.ctx, SCALE, splits, ws,
                                    self.k_ts, self.v_ts, empty, error_flag)

    def check(self, o, lse, empty=None):
        o, lse = o.double().cpu().numpy(), lse.double().cpu().numpy()
        assert o.shape == (len(self.ctxs), self.H, self.W) and lse.shape == (self.H, len(self.ctxs))
        for t, (k, v) in enumerate(self.rows):
            if empty is not None and empty[t]:
                k, v = k[:0], v[:0]
            eo, el, av, aq = ref.attention(self.q[t], k, v, SCALE)
            if k.shape[0] == 0:
                assert (o[t] == 0).all() and np.isneginf(lse[:, t]).all()
                continue
            d = (self.W / 16 + 8) * U32 * aq
            tol = ((U16 + 2 * d[:, None] + (k.shape[0] / 16 + 8) * U32) * av * 1.01 + U16 * 1.01 * np.abs(eo)
                   + 2.0 ** -36 * np.abs(v).sum(0))
            assert (np.abs(o[t] - eo) <= tol).all(), (t, np.abs(o[t] - eo).max(), (np.abs(o[t] - eo) / tol).max())
            assert (np.abs(lse[:, t] - el) <= d + 8 * U32 * (1 + np.abs(el)) + (k.shape[0] / 16 + 8) * U32).all(), t


EDGES = [0, 1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 0, 300, 1029]


@pytest.mark.parametrize('W', [256, 512, 1024])
@pytest.mark.parametrize('page', [16, 32, 48])
def test_history_edge_lengths(W, page):
    h = History(EDGES, W=W, page=page, seed=W + page)
    h.check(*h.run())


@pytest.mark.parametrize('H', [1, 2, 7, 8, 9, 15, 16])
def test_history_head_counts(H):
    h = History([0, 5, 130, 700], H=H, seed=H)
    h.check(*h.run())


@pytest.mark.parametrize('ctxs', [[1], [40], [128], [5000], [0], [0, 0, 0]])
@pytest.mark.parametrize('W', [256, 512])
def test_history_single_requests(W, ctxs):
    h = History(ctxs, W=W, seed=len(ctxs) + ctxs[0])
    h.check(*h.run(splits=64))


@pytest.mark.parametrize('splits', [1, 2, 3, 16, 296])
def test_history_split_counts(splits):
    h = History([900, 3, 0, 257, 64], seed=splits)
    h.check(*h.run(splits=splits))


def test_history_many_rows_take_one_cta_each():
    rng = np.random.default_rng(5)
    h = History(rng.integers(0, 40, 1100).tolist(), W=256, H=3, seed=5)
    h.check(*h.run(splits=2))


def test_history_strided_inputs_and_padded_blocks():
    h = History([33, 0, 200], H=4, seed=9, pad=16 * 7)
    big = torch.full((3, 9, 1024), float('nan'), dtype=BF16, device=CUDA)
    q = big[:, 1:9:2, 256:768]
    q.copy_(h.qd)
    h.check(*h.run(q=q))


def test_history_empty_flags_and_dtypes():
    h = History([50, 20, 0, 64], seed=3)
    for dtype in (torch.bool, torch.uint8, torch.int32):
        e = torch.tensor([0, 1, 0, 1], device=CUDA).to(dtype)
        h.check(*h.run(empty=e), empty=[0, 1, 0, 1])


def test_history_large_scores_and_values():
    """Peaked softmax: scores of thousands (one key takes all), values up to 7 * 448 * 2^6."""
    h = History([200, 17], seed=11, k_ts=64.0, v_ts=64.0)
    h.check(*h.run())


def test_history_block_outside_the_cache_reads_as_zeros():
    h = History([40, 100], seed=4)
    for bad in (-1, h.cache.shape[0], 2 ** 30):
        h.bt[1, 2] = bad
        k, v = (x.copy() for x in h.rows[1])
        k[32:48], v[32:48] = 0, 0
        h.rows[1] = (k, v)
        flag = torch.zeros(1, dtype=torch.int32, device=CUDA)
        h.check(*h.run(error_flag=flag))
        assert flag.item() == pkg('_lib').ERR_BLOCK


def test_history_context_longer_than_its_table_reads_zeros():
    h = History([64], seed=6)
    h.bt = h.bt[:, :3].contiguous()
    k, v = (x.copy() for x in h.rows[0])
    k[48:], v[48:] = 0, 0
    h.rows[0] = (k, v)
    flag = torch.zeros(1, dtype=torch.int32, device=CUDA)
    h.check(*h.run(error_flag=flag))
    assert flag.item() == pkg('_lib').ERR_BLOCK


def test_history_is_what_s6_ops_runs_for_a_uint8_cache():
    ops = pkg('s6_ops')
    h = History([70, 0, 300], seed=8)
    o, lse = ops.history_attention(h.qd, h.cache, h.bt, h.ctx, SCALE, 8, ops.S6Workspace(h.H, h.W, 24), h.k_ts, h.v_ts,
                                   'b200')
    h.check(o, lse)
    a, b = h.run()
    assert torch.equal(o, a) and torch.equal(lse, b)


def test_history_repeats_bit_for_bit_and_in_a_graph():
    h = History([1000, 40, 0, 333], seed=12)
    ops = pkg('s6_ops')
    ws = ops.S6Workspace(h.H, h.W, 4 * 8)
    a = h.run(ws=ws)
    b = h.run(ws=ws)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        h.run(ws=ws)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = h.run(ws=ws)
    # new queries, lengths, tables and cache contents behind the same addresses
    other = History([333, 0, 990, 1], seed=13)
    n = other.cache.shape[0]
    wide = min(h.bt.shape[1], other.bt.shape[1])
    assert n <= h.cache.shape[0] and wide * 16 >= 990
    h.qd.copy_(other.qd)
    h.cache[:n].copy_(other.cache)
    h.bt[:, :wide].copy_(other.bt[:, :wide])
    h.ctx.copy_(other.ctx)
    graph.replay()
    other.check(*out)


def test_history_on_two_streams_with_their_own_workspaces():
    a, b = History([2000, 10], seed=14), History([50, 1500], seed=15)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], []
    for s, h in zip(streams, (a, b)):
        with torch.cuda.stream(s):
            got.append([h.run() for _ in range(5)][-1])
    torch.cuda.synchronize()
    a.check(*got[0])
    b.check(*got[1])


# ------------------------------------------------------------------------------------ commit and gather
def commit_setup(share, W, page, seed, start=None, padding=0):
    rng = np.random.default_rng(seed)
    R, T = len(share), sum(share) + padding
    start = start or [0] * R
    pages = [-(-(s + n) // page) for s, n in zip(start, share)]
    nb = sum(pages) + 1
    perm = (rng.permutation(nb - 1) + 1).astype(np.int32)
    bt = np.zeros((R, max(pages + [1])), dtype=np.int32)
    at = 0
    for r, n in enumerate(pages):
        bt[r, :n] = perm[at:at + n]
        at += n
    pos = np.concatenate([np.arange(s, s + n) for s, n in zip(start, share)] + [np.arange(padding)]).astype(np.int64)
    qsl = np.concatenate(([0], np.cumsum(share))).astype(np.int32)
    req = np.repeat(np.arange(R), share)
    slots = np.full(T, -1, dtype=np.int64)
    slots[:len(req)] = bt[req, pos[:len(req)] // page].astype(np.int64) * page + pos[:len(req)] % page
    maxpos = max(int(pos.max()) + 1, 1) if T else 1
    ang = np.arange(maxpos)[:, None] * (10000.0 ** (-2 * (np.arange(W // 2) % 64) / 128))
    table = ref.bf16(np.concatenate((np.cos(ang), np.sin(ang)), 1))
    row = bf(rng, T, 2 * W) * np.exp2(rng.integers(-3, 4, (T, 2 * W)))
    row = ref.bf16(row)
    return dict(row=row, pos=pos, table=table, bt=bt, qsl=qsl, slots=slots, nb=nb)


COMMITS = [([1], 512, 16, 0), ([1, 1, 1], 256, 16, 0), ([5, 0, 17, 1], 512, 16, 3), ([40, 33], 1024, 32, 0),
           ([7], 256, 48, 2), ([64] * 3, 512, 32, 1), ([1] * 130, 512, 16, 5),
           ([4000, 1, 5601], 1024, 16, 7)]    # enough tokens for several rows a thread


@pytest.mark.parametrize('share,W,page,padding', COMMITS)
def test_commit_is_exact_and_touches_its_own_rows_alone(share, W, page, padding):
    q4 = pkg('q4')
    c = commit_setup(share, W, page, seed=sum(share) + W, padding=padding, start=[3 * i for i in range(len(share))])
    rng = np.random.default_rng(1)
    before = rng.integers(0, 256, (c['nb'], 1, page, 17 * W // 16)).astype(np.uint8)
    want = before.copy()
    k_ts, v_ts = 0.25, 2.0
    rotated = ref.rope(c['row'][:, :W], c['table'], c['pos'])
    for t, s in enumerate(c['slots']):
        if s >= 0:
            ref.put_row(want, W, page, int(s), rotated[t], c['row'][t, W:], k_ts, v_ts)
    cache = dev(before)
    slots = q4.commit_rows(dev(c['row'], BF16), dev(c['pos']), dev(c['table'], BF16), cache, dev(c['bt']),
                           dev(c['qsl']), k_ts, v_ts)
    assert slots.tolist() == c['slots'].tolist()
    assert np.array_equal(cache.cpu().numpy(), want)
    got = q4.gather_slots(cache, slots, k_ts, v_ts).double().cpu().numpy()
    for t, s in enumerate(c['slots']):
        e = np.zeros(2 * W) if s < 0 else np.concatenate((ref.stored(rotated[t], k_ts), ref.stored(c['row'][t, W:], v_ts)))
        assert np.array_equal(got[t], e), t


def test_commit_extreme_rows():
    """Zeros, tiny and huge values, infinities; a scale that underflows stores zeros, one that saturates clamps."""
    q4 = pkg('q4')
    W, page = 256, 16
    c = commit_setup([6], W, page, seed=0)
    row = np.zeros((6, 2 * W))
    row[1] = 2.0 ** -20
    row[2] = ref.bf16(np.linspace(-1e5, 1e5, 2 * W))
    row[3, 7], row[3, W + 40] = 1.0, -3.0
    row[4] = ref.bf16(np.linspace(0, 2.0 ** -7, 2 * W))        # scales in e4m3's subnormal range
    row[5, W + 3], row[5, W + 4] = np.inf, -np.inf
    c['table'][:, :W // 2], c['table'][:, W // 2:] = 1, 0      # the identity rotation
    cache = q4.new_cache(c['nb'], page, W)
    slots = q4.commit_rows(dev(row, BF16), dev(c['pos']), dev(c['table'], BF16), cache, dev(c['bt']), dev(c['qsl']))
    got = q4.gather_slots(cache, slots).double().cpu().numpy()
    for t in range(5):
        assert np.array_equal(got[t], np.concatenate((ref.stored(row[t, :W], 1.0), ref.stored(row[t, W:], 1.0)))), t
    assert got[5, W + 3] == 7 * 448 and got[5, W + 4] == -7 * 448 and (np.delete(got[5], [W + 3, W + 4]) == 0).all()


def test_commit_tensor_scales_that_are_not_powers_of_two():
    """3 / 8 and 5: steps of at most 7 significant bits, exact in fp32, so the codes are the formula's.  (No amax of 8
    bits lies half way between two normal scales: 21 / 8 and 35 times an odd number of 5 bits has more than 8.)"""
    q4 = pkg('q4')
    c = commit_setup([70, 3], 512, 16, seed=4, start=[0, 9])
    rotated = ref.rope(c['row'][:, :512], c['table'], c['pos'])
    want = np.zeros((c['nb'], 1, 16, 544), dtype=np.uint8)
    for t, s in enumerate(c['slots']):
        ref.put_row(want, 512, 16, int(s), rotated[t], c['row'][t, 512:], 0.375, 5.0)
    cache = dev(np.zeros_like(want))
    q4.commit_rows(dev(c['row'], BF16), dev(c['pos']), dev(c['table'], BF16), cache, dev(c['bt']), dev(c['qsl']), 0.375, 5.0)
    assert np.array_equal(cache.cpu().numpy(), want)


def test_commit_skips_positions_without_a_block():
    q4 = pkg('q4')
    W, page = 256, 16
    c = commit_setup([6], W, page, seed=2)
    pos = c['pos'].copy()
    pos[1], pos[2] = -1, 10 ** 12                              # before the first row, past the table
    bt = np.array([[1]], dtype=np.int32)
    cache = q4.new_cache(c['nb'], page, W)
    slots = q4.commit_rows(dev(c['row'], BF16), dev(pos), dev(c['table'], BF16), cache, dev(bt), dev(c['qsl']))
    assert slots.tolist() == [16, -1, -1, 19, 20, 21]
    for bad in (-1, c['nb'], 2 ** 30):
        slots = q4.commit_rows(dev(c['row'], BF16), dev(c['pos']), dev(c['table'], BF16), cache.clone(),
                               dev(np.array([[bad]], dtype=np.int32)), dev(c['qsl']))
        assert slots.tolist() == [-1] * 6


def test_commit_strided_rows_and_padded_blocks():
    q4 = pkg('q4')
    W, page = 512, 16
    c = commit_setup([9, 20], W, page, seed=4)
    T, nb, size = 29, c['nb'], page * 17 * W // 16
    wide = torch.full((T, 2 * W + 24), float('nan'), dtype=BF16, device=CUDA)
    wide[:, 8:8 + 2 * W] = dev(c['row'], BF16)
    full = torch.full((nb, size + 160), 77, dtype=torch.uint8, device=CUDA)
    cache = full.as_strided((nb, 1, page, 17 * W // 16), (full.stride(0), size, 17 * W // 16, 1))
    args = dev(c['pos']), dev(c['table'], BF16)
    slots = q4.commit_rows(wide[:, 8:8 + 2 * W], *args, cache, dev(c['bt']), dev(c['qsl']), 0.5, 0.5)
    plain = torch.full((nb, 1, page, 17 * W // 16), 77, dtype=torch.uint8, device=CUDA)
    q4.commit_rows(dev(c['row'], BF16), *args, plain, dev(c['bt']), dev(c['qsl']), 0.5, 0.5)
    assert torch.equal(cache, plain) and (full[:, size:] == 77).all()
    out = torch.full((T, 2 * W + 40), 5.0, dtype=BF16, device=CUDA)
    got = q4.gather_slots(cache, slots, 0.5, 0.5, out=out[:, 8:8 + 2 * W])
    assert torch.equal(got, q4.gather_slots(plain, slots, 0.5, 0.5))
    assert (out[:, :8] == 5).all() and (out[:, 8 + 2 * W:] == 5).all()


@pytest.mark.parametrize('W,page,length', [(256, 16, 1), (256, 32, 33), (512, 16, 0), (512, 48, 100), (1024, 16, 250),
                                           (512, 16, 16), (256, 48, 4097), (512, 16, 4200), (1024, 16, 4111)])
def test_gather_rows_is_exact(W, page, length):
    q4 = pkg('q4')
    rng = np.random.default_rng(length)
    n = -(-length // page)
    cache, k, v = ref.random_cache(rng, n + 3, page, W)
    blocks = (rng.permutation(n + 2) + 1)[:n + 1].astype(np.int32)      # one entry more than the rows need
    got = q4.gather_rows(dev(cache), dev(blocks), length, 0.5, 4.0).double().cpu().numpy()
    want = np.concatenate((k[blocks[:n]].reshape(-1, W)[:length] * 0.5, v[blocks[:n]].reshape(-1, W)[:length] * 4), 1)
    assert np.array_equal(got, want)


@pytest.mark.parametrize('k_ts,v_ts', [(0.3, 7.0), (2.0 ** -120, 2.0 ** 110), (0.375, 2.0 ** -100)])
def test_gather_tensor_scales(k_ts, v_ts):
    """Any tensor scale: the exact (n - 8) s times the fp32 scale, rounded to fp32 and to bf16; in range, a power of two
    of any size is exact."""
    q4 = pkg('q4')
    rng = np.random.default_rng(5)
    cache, k, v = ref.random_cache(rng, 3, 16, 256)
    got = q4.gather_rows(dev(cache), dev(np.array([2, 0], dtype=np.int32)), 30, k_ts, v_ts).double().cpu().numpy()
    for half, x, ts in ((got[:, :256], k, k_ts), (got[:, 256:], v, v_ts)):
        want = ref.bf16((x[[2, 0]].reshape(-1, 256)[:30].astype(np.float32) * np.float32(ts)).astype(np.float64))
        assert np.array_equal(half, want)


def test_gather_block_outside_the_cache():
    q4 = pkg('q4')
    rng = np.random.default_rng(0)
    cache, k, v = ref.random_cache(rng, 3, 16, 256)
    for bad in (-1, 3, 2 ** 30):
        flag = torch.zeros(1, dtype=torch.int32, device=CUDA)
        got = q4.gather_rows(dev(cache), dev(np.array([2, bad, 1], dtype=np.int32)), 48, error_flag=flag)
        got = got.double().cpu().numpy()
        assert np.array_equal(got[:16, :256], k[2]) and (got[16:32] == 0).all() and np.array_equal(got[32:, 256:], v[1])
        assert flag.item() == pkg('_lib').ERR_BLOCK
    flag = torch.zeros(1, dtype=torch.int32, device=CUDA)
    got = q4.gather_slots(dev(cache), dev(np.array([-1, 47, 48, 5], dtype=np.int64)), error_flag=flag)
    got = got.double().cpu().numpy()
    assert (got[0] == 0).all() and np.array_equal(got[1, :256], k[2, 15]) and (got[2] == 0).all()
    assert np.array_equal(got[3, 256:], v[0, 5]) and flag.item() == pkg('_lib').ERR_BLOCK


def test_round_trip_error_is_half_a_step():
    """What comes back is off by at most half a step, plus what the scale's own rounding (2^-4) can clip: the
    largest value is 7 (1 + 2^-4) = 7.4375 steps at most, still within half a step of 7."""
    q4 = pkg('q4')
    W, page = 512, 16
    c = commit_setup([64], W, page, seed=7)
    cache = q4.new_cache(c['nb'], page, W)
    slots = q4.commit_rows(dev(c['row'], BF16), dev(c['pos']), dev(c['table'], BF16), cache, dev(c['bt']), dev(c['qsl']))
    got = q4.gather_slots(cache, slots).double().cpu().numpy()
    v = c['row'][:, W:].reshape(64, -1, 32)
    amax = np.abs(v).max(-1, keepdims=True)
    assert (amax > 0.2).all()
    assert (np.abs(got[:, W:].reshape(v.shape) - v) <= amax / 7 * (1 + 2.0 ** -4) / 2).all()


# ------------------------------------------------------------------------------------ linear
LINEARS = [(1, 16, 32), (1, 1, 128), (3, 17, 160), (8, 100, 96), (9, 2048, 2048), (16, 33, 1024), (17, 48, 4096),
           (33, 512, 2048), (64, 1024, 128), (65, 250, 416), (127, 64, 2048), (128, 256, 128), (130, 512, 2048),
           (257, 1024, 512), (300, 272, 192), (200, 100, 320), (1, 6144, 2048), (600, 768, 640),
           (5, 8200, 64), (64, 2048, 160), (57, 2030, 96), (40, 5000, 64), (31, 5000, 64)]


def linear_case(T, N, K, seed):
    rng = np.random.default_rng(seed)
    w = bf(rng, N, K, std=K ** -0.5)
    x = bf(rng, T, K) * np.exp2(rng.integers(-2, 3, (T, K)))
    return ref.bf16(x), w, bf(rng, T, N)


def check_linear(y, x, wq, scale, res, K):
    exact = x @ wq.T * scale
    mass = np.abs(x) @ np.abs(wq).T * scale
    tol = (K / 16 + 8) * U32 * mass
    if res is not None:
        exact = exact + res
    y = y.double().cpu().numpy()
    tol = tol * (1 + U16) + U16 * 1.01 * np.abs(exact) + 1e-30
    assert (np.abs(y - exact) <= tol).all(), (np.abs(y - exact) / tol).max()


@pytest.mark.parametrize('T,N,K', LINEARS)
@pytest.mark.parametrize('residual', [False, True])
def test_linear(T, N, K, residual):
    q4 = pkg('q4')
    x, w, res = linear_case(T, N, K, seed=T + N + K)
    packed, scale = q4.quantize_weight(dev(w, BF16))
    n, b = ref.quantize(w, scale)
    wq = (n - 8) * np.repeat(ref.E4M3[b], 32, -1)
    assert np.array_equal(ref.unpack_weight(packed.cpu().numpy(), N, K), wq)      # quantised and packed exactly
    y = q4.linear(dev(x, BF16), packed, N, scale, dev(res, BF16) if residual else None)
    check_linear(y, x, wq, scale, res if residual else None, K)


# enough tiles for the kernel of the largest calls: ends inside a tile in every direction, the shortest K, one block of K
# more than a whole number of stages, and rows of outputs that are not 16-byte aligned
@pytest.mark.parametrize('T,N,K', [(1030, 2001, 416), (4096, 512, 128), (8200, 130, 32), (2100, 1000, 2048),
                                   (1025, 1800, 832), (4000, 400, 64)])
@pytest.mark.parametrize('residual', [False, True])
def test_linear_wide(T, N, K, residual):
    test_linear(T, N, K, residual)


@pytest.mark.parametrize('T', [2, 20, 300])
def test_linear_strides_in_place_residual_and_zero_tokens(T):
    q4 = pkg('q4')
    N, K = 256, 384
    x, w, res = linear_case(T, N, K, seed=T)
    packed, scale = q4.quantize_weight(dev(w, BF16), 0.0078125)
    wq = ref.unpack_weight(packed.cpu().numpy(), N, K)
    xs = torch.full((T, K + 40), float('nan'), dtype=BF16, device=CUDA)
    xs[:, 16:16 + K] = dev(x, BF16)
    stream = torch.full((T, N + 24), 3.0, dtype=BF16, device=CUDA)
    y = stream[:, 8:8 + N]
    y.copy_(dev(res, BF16))
    got = q4.linear(xs[:, 16:16 + K], packed, N, scale, residual=y, out=y)
    assert got.data_ptr() == y.data_ptr()
    check_linear(y, x, wq, scale, res, K)
    assert (stream[:, :8] == 3).all() and (stream[:, 8 + N:] == 3).all()
    none = q4.linear(xs[:0, 16:16 + K], packed, N, scale)
    assert none.shape == (0, N)


def test_linear_odd_output_strides():
    """A residual and an output whose rows are not 4-byte aligned."""
    q4 = pkg('q4')
    for T in (5, 140):
        N, K = 96, 256
        x, w, res = linear_case(T, N, K, seed=T)
        packed, scale = q4.quantize_weight(dev(w, BF16))
        wq = ref.unpack_weight(packed.cpu().numpy(), N, K)
        base = torch.zeros(T, N + 3, dtype=BF16, device=CUDA)
        y, r = base[:, 1:1 + N], torch.zeros(T, N + 1, dtype=BF16, device=CUDA)[:, 1:]
        r.copy_(dev(res, BF16))
        q4.linear(dev(x, BF16), packed, N, scale, r, out=y)
        check_linear(y, x, wq, scale, res, K)
        assert (base[:, 0] == 0).all() and (base[:, 1 + N:] == 0).all()


def test_linear_large_inputs_and_graph_replay():
    q4 = pkg('q4')
    N, K = 128, 512
    for T in (4, 256):
        x, w, _ = linear_case(T, N, K, seed=T)
        x = ref.bf16(x * 2.0 ** 40)                              # beyond fp16's range
        packed, scale = q4.quantize_weight(dev(w, BF16))
        wq = ref.unpack_weight(packed.cpu().numpy(), N, K)
        xd = torch.zeros(T, K, dtype=BF16, device=CUDA)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            q4.linear(xd, packed, N, scale)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = q4.linear(xd, packed, N, scale)
        xd.copy_(dev(x, BF16))
        graph.replay()
        check_linear(y, x, wq, scale, None, K)


def test_linear_non_finite_inputs_stay_in_their_row():
    q4 = pkg('q4')
    for T in (6, 200):
        x, w, _ = linear_case(T, 64, 256, seed=T)
        packed, scale = q4.quantize_weight(dev(w, BF16))
        wq = ref.unpack_weight(packed.cpu().numpy(), 64, 256)
        xd = dev(x, BF16)
        xd[2] = float('nan')
        xd[4, 5] = float('inf')
        y = q4.linear(xd, packed, 64, scale)
        assert torch.isnan(y[2]).all() and not torch.isfinite(y[4]).all()
        keep = [t for t in range(T) if t not in (2, 4)]
        check_linear(y[keep], x[keep], wq, scale, None, 256)
