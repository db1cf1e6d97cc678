"""The 4-bit operators together, as a serving step uses them: ``ouro_attention.LatentAttention.forward`` with 4-bit
latent caches, packed QKV / output weights and packed writers, over prefill, decode, mixed and padded steps.

Per step and loop:

* the projections, the writer state and the output are ``q4.linear``'s, whose own error is bounded in test_q4_gpu;
* the committed rows are the float64 restatement's, exactly, and no other row of the cache changes;
* the attention equals the bf16 path's over a bf16 cache that holds the same values (they are exact in bf16).

The attention's bound.  Both sides take the same exact part and the same values, so they differ by the two readers'
errors alone.  With d = (W / 16 + 8) 2^-22 sum|q k| scale, each reader moves p by a factor exp(+-2 d), rounds p
(2^-8), the latent result (2^-8) and the projected one (2^-8): two readers make 6 2^-8 + 8 d of S = sum_r |B| sum p|v|.
The share of the latent part moves by a factor exp(+-2 d) between them, which is worth 2 d (S + |exact part|), the
latter at most the largest |v|; the two results are rounded (2 2^-8 |o|).  B picks columns here (one +-1 per output),
so that S is one column's sum p|v| and not 512 of them.  Small p (2^-36 sum|v|, see test_q4_gpu): below 2^-30 here.
"""
import numpy as np
import pytest
import torch

import q4_reference as ref
from conftest import pkg

pytestmark = pytest.mark.gpu
CUDA, BF16, I32 = 'cuda', torch.bfloat16, torch.int32
THETA, MAXPOS, LOOPS, D = 1e6, 512, 4, 128
U16, U32 = 2.0 ** -8, 2.0 ** -22


class Layer:
    def __init__(self, H, hidden, rank, rank1, window, page, seed, nb=40, main_scale=(0.03125, 0.0625),
                 l1_scale=(0.0625, 0.03125)):
        oa, lay, lat, q4 = pkg('ouro_attention'), pkg('s6_layer'), pkg('latent'), pkg('q4')
        self.g = torch.Generator(device=CUDA).manual_seed(seed)
        self.H, self.hidden, self.window, self.page, self.nb = H, hidden, window, page, nb
        self.widths = [rank1] + [rank] * (LOOPS - 1)
        sl = lat.LatentLayer(hidden, H, D, LOOPS, rank, rank, rank1).to(CUDA, BF16).requires_grad_(False)
        with torch.no_grad():
            for p in (sl.q_absorb, sl.q_absorb1):
                p.copy_(self.rnd(*p.shape, std=D ** -0.5))
            for p in (sl.out_absorb, sl.out_absorb1):                 # [.., rank, D]: output column i is +-latent column
                p.zero_()
                flat = p.view(-1, *p.shape[-2:])
                for h in range(flat.shape[0]):
                    cols = torch.randperm(p.shape[-2], generator=self.g, device=CUDA)[:D]
                    flat[h, cols, torch.arange(D, device=CUDA)] = torch.where(torch.rand(D, generator=self.g, device=CUDA)
                                                                              < 0.5, -1.0, 1.0).to(BF16)
            for lin in (*sl.cand_s, sl.cand1):
                lin.weight.copy_(self.rnd(*lin.weight.shape, std=hidden ** -0.5))
        sl.pack_writers()
        self.sl = sl
        self.qkv = q4.Weight.of(self.rnd(3 * H * D, hidden, std=hidden ** -0.5))
        self.o = q4.Weight.of(self.rnd(hidden, H * D, std=(H * D) ** -0.5))
        inv = lay.latent_inv_freq(D, THETA)
        self.tables = {w: lay.latent_rope_table(MAXPOS, inv, w, BF16).to(CUDA) for w in set(self.widths)}
        ang = torch.arange(MAXPOS).float()[:, None] * inv[None]
        self.attn = oa.LatentAttention(sl, self.qkv, self.o, torch.cat((ang.cos(), ang.sin()), -1).to(CUDA), window)
        self.caches = oa.PagedCaches(
            main=self.poisoned(rank), l1=self.poisoned(rank1), latent_table=None,
            exact=[torch.full((nb, page, H, 2 * D), float('nan'), dtype=BF16, device=CUDA) for _ in range(LOOPS)],
            exact_table=None, main_scale=main_scale, l1_scale=l1_scale)
        # the same histories in bf16 caches
        self.bf16 = [torch.full((nb, 1, page, 2 * w), float('nan'), dtype=BF16, device=CUDA) for w in (rank1, rank)]
        self.rng = np.random.default_rng(seed)
        self.free = (self.rng.permutation(nb - 1) + 1).tolist()
        self.blocks, self.length = {}, {}

    def rnd(self, *shape, std=1.0):
        return (torch.randn(*shape, generator=self.g, device=CUDA) * std).to(BF16)

    def poisoned(self, width):
        """Every byte 0x7f: codes 7 and 15, scales NaN."""
        cache = pkg('q4').new_cache(self.nb, self.page, width)
        return cache.fill_(0x7f)

    def step(self, requests, padded_requests=0, padding_tokens=0, splits=4):
        """Metadata of one step: ``(ctx, query_start_loc, slots, contexts)``."""
        ops, lay = pkg('s6_ops'), pkg('s6_layer')
        counts = [n for _, n in requests]
        before = [self.length.get(r, 0) for r, _ in requests]
        real, R = sum(counts), len(requests) + padded_requests
        T = real + padding_tokens
        starts = np.concatenate(([0], np.cumsum(counts)))
        qsl = np.concatenate((starts, [real] * padded_requests)).astype(np.int32)
        seq = np.array([c + n for c, n in zip(before, counts)] + [0] * padded_requests, dtype=np.int32)
        pos = np.concatenate([np.arange(c, c + n) for c, n in zip(before, counts)] + [np.ones(padding_tokens)]).astype(np.int64)
        table = self.rng.integers(1, self.nb, (R, 8)).astype(np.int32)       # stale columns name live blocks
        for i, (r, n) in enumerate(requests):
            own = self.blocks.setdefault(r, [])
            while len(own) * self.page < before[i] + n:
                own.append(self.free.pop())
            table[i, :len(own)] = own
            self.length[r] = before[i] + n
        self.caches.latent_table = self.caches.exact_table = torch.from_numpy(table).to(CUDA)
        ws = ops.S6Workspace(self.H, max(self.widths), max(T, 1) * splits)
        ctx = lay.StepContext(torch.from_numpy(pos).to(CUDA), torch.from_numpy(qsl).to(CUDA), torch.from_numpy(seq).to(CUDA),
                              max(counts), T, self.tables, D ** -0.5, ops.B200_BACKENDS, ws, splits, window=self.window)
        request = np.repeat(np.arange(len(counts)), counts)
        slots = table[request, pos[:real] // self.page].astype(np.int64) * self.page + pos[:real] % self.page
        return ctx, slots, pos, table[request], np.repeat(before, counts)

    def run(self, requests, **kw):
        q4, lay = pkg('q4'), pkg('s6_layer')
        ctx, slots, pos, tables, before = self.step(requests, **kw)
        T, real, H = ctx.positions.shape[0], len(slots), self.H
        state = None
        for loop in range(LOOPS):
            width = self.widths[loop]
            cache, scales = (self.caches.l1, self.caches.l1_scale) if loop == 0 else (self.caches.main, self.caches.main_scale)
            hidden = self.rnd(T, self.hidden)
            was = cache.clone()
            previous = None if state is None else state.reg
            out, state, attn = self.attn.forward(ctx.positions, hidden, loop, state, ctx, self.caches, return_attention=True)
            # projections and the writer: the 4-bit linear's own results
            assert torch.equal(out, self.o.linear(attn.reshape(T, H * D)))
            row = state.first if loop == 0 else state.reg
            assert torch.equal(row, self.sl.packed_writers[loop].linear(hidden, previous))
            # the attention, against the bf16 path over the same values
            qkv = self.qkv.linear(hidden)
            q, k, v = (x.view(T, H, D) for x in qkv.split(H * D, -1))
            q_lat = ctx.latent_query(self.sl, loop, q)
            k_rope, window = torch.empty(T, H, D, dtype=BF16, device=CUDA), None
            if self.window:
                cache_e = self.caches.exact[loop].transpose(1, 2)
                window = (cache_e, self.caches.exact_table)
                self.attn._exact_append(q, k, v, k_rope, ctx.positions, *window, ctx)
            else:
                self.attn._exact_append(q, k, v, k_rope, ctx.positions, None, None, ctx)
            same = self.bf16[min(loop, 1)]
            want = lay.attend(self.sl, loop, q_lat, q, k_rope, v, same, self.caches.latent_table, None, None, ctx, window)
            got, want = attn.double().cpu().numpy(), want.double().cpu().numpy()
            assert (got[real:] == 0).all() and np.isfinite(got).all()
            bound = self.bound(loop, q_lat, tables, before, v, np.abs(want[:real]))
            err = np.abs(got[:real] - want[:real])
            assert (err <= bound).all(), (loop, float((err / bound).max()))
            # the committed rows
            if loop not in (0, LOOPS - 1):
                assert torch.equal(cache, was)
                continue
            expect = was.cpu().numpy()
            values = row.double().cpu().numpy()[:real]
            key = ref.rope(values[:, :width], self.tables[width].double().cpu().numpy(), pos[:real])
            for t in range(real):
                ref.put_row(expect, width, self.page, slots[t], key[t], values[t, width:], *scales)
            np.testing.assert_array_equal(cache.cpu().numpy(), expect)
            at = torch.from_numpy(slots).to(CUDA)
            same.view(-1, 2 * width)[at] = q4.gather_slots(cache, at, *scales)
            stored = np.concatenate((ref.stored(key, scales[0]), ref.stored(values[:, width:], scales[1])), 1)
            np.testing.assert_array_equal(same.view(-1, 2 * width)[at].double().cpu().numpy(), stored)
        return ctx

    def bound(self, loop, q_lat, tables, before, v, o):
        """The docstring's bound for the real tokens ``[real, H, D]``."""
        W, scale = self.widths[loop], D ** -0.5
        B = np.abs(self.sl.readers(loop)[1].double().cpu().numpy())          # [H, W, D]
        rows = self.bf16[min(loop, 1)].double().cpu().numpy().reshape(-1, 2 * W)
        q, vmax = q_lat.double().cpu().numpy(), float(v.abs().max())
        out = np.zeros_like(o)
        for t in range(len(before)):
            n = max(0, before[t] - self.window)
            i = np.arange(n)
            r = rows[tables[t, i // self.page].astype(np.int64) * self.page + i % self.page]
            _, _, pv, sumqk = ref.attention(q[t], r[:, :W], r[:, W:], scale)
            d = ((W / 16 + 8) * U32 * sumqk)[:, None]
            S = np.einsum('hw,hwd->hd', pv, B)
            out[t] = S * (6 * U16 + 8 * d) + 2 * d * (S + vmax) + 2 * U16 * o[t] + 2.0 ** -30
        return out


@pytest.mark.parametrize('H,hidden,rank,rank1,window,page', [(16, 2048, 512, 256, 32, 16), (5, 416, 256, 256, 7, 32),
                                                           (2, 256, 512, 512, 16, 16)])
def test_serving_steps(H, hidden, rank, rank1, window, page):
    layer = Layer(H, hidden, rank, rank1, window, page, seed=H)
    layer.run([(0, 40)])                                                     # full-prompt prefill
    layer.run([(0, 1)])                                                      # decode
    layer.run([(1, 33), (2, 70)])
    layer.run([(0, 1), (1, 1), (2, 1)], padded_requests=1, padding_tokens=2)
    layer.run([(1, 17), (3, 5), (0, 1)])                                     # prefill and decode together
    layer.run([(3, 1), (2, 1), (0, 1)], padding_tokens=1, splits=1)
    # what a finished request leaves: its rows as the exporter reads them
    ce, q4, c = pkg('cache_export'), pkg('q4'), layer.caches
    blocks, n = layer.blocks[2], layer.length[2]
    rows, = ce.export_rows([c.main], [c.l1], blocks, blocks, n, page, main_scales=[c.main_scale], l1_scales=[c.l1_scale])
    at = torch.tensor(blocks, device=CUDA).repeat_interleave(page)[:n] * page + torch.arange(n, device=CUDA) % page
    want = torch.cat([s.view(-1, s.shape[-1])[at] for s in (layer.bf16[1], layer.bf16[0])], 1)
    assert torch.equal(rows[0], want.cpu())
    with pytest.raises(IndexError, match='outside'):
        ce.export_rows([c.main], [c.l1], [layer.nb] + blocks, blocks, n, page)
    with pytest.raises(ValueError, match='per layer'):
        ce.export_rows([c.main], [c.l1], blocks, blocks, n, page, main_scales=[])


def test_windowless_steps():
    layer = Layer(4, 512, 512, 256, 0, 16, seed=3)
    layer.run([(0, 20), (1, 3)])
    layer.run([(0, 1), (1, 9)], padding_tokens=1)
    layer.run([(0, 1), (1, 1)])


def test_decode_step_replays_from_a_graph():
    """All loops of a decode step in one CUDA graph: the eager step's bits, for new inputs too."""
    layer = Layer(16, 2048, 512, 256, 32, 16, seed=9)
    layer.run([(0, 100), (1, 41)])
    ctx, slots, *_ = layer.step([(0, 1), (1, 1)], padding_tokens=2)
    T, c = ctx.positions.shape[0], layer.caches
    hidden = [layer.rnd(T, layer.hidden) for _ in range(LOOPS)]
    ctx.block_table(c.latent_table), ctx.block_table(c.exact_table)

    def all_loops():
        state, outs = None, []
        for loop in range(LOOPS):
            out, state = layer.attn.forward(ctx.positions, hidden[loop], loop, state, ctx, c)
            outs.append(out)
        return outs

    begin = [x.clone() for x in (c.main, c.l1, *c.exact)]

    def restore():
        for x, b in zip((c.main, c.l1, *c.exact), begin):
            x.copy_(b)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        all_loops()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = all_loops()
    for trial in range(3):
        for h in hidden:
            h.copy_(layer.rnd(T, layer.hidden))
        restore()
        graph.replay()
        got = [o.clone() for o in outs] + [c.main.clone(), c.l1.clone()]
        restore()
        want = all_loops() + [c.main, c.l1]
        assert all(torch.equal(a, b) for a, b in zip(got, want)), trial
        # the rows behind the tables' lengths stay as they were, all but the two committed ones
        moved = (c.main.cpu() != begin[0].cpu()).flatten(2).any(-1).flatten()
        same_page = set((slots // layer.page).tolist())
        assert set(moved.nonzero().flatten().tolist()) <= same_page


def test_a_1024_wide_latent_is_refused_by_the_combine():
    """``s6_layer.attend`` takes latents of 256 and 512, of either kind of cache (the reader alone takes 1024 too)."""
    layer = Layer(2, 256, 1024, 512, 16, 16, seed=2)
    with pytest.raises(ValueError, match='width 1024 unsupported'):
        layer.run([(0, 40)])
