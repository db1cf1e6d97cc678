"""The 4-bit operators' host side, without a GPU: the format's arithmetic, the refusals of ``q4`` and of the C
entry points behind it (all before any device work), and the geometry checks."""
import ctypes
import math

import numpy as np
import pytest
import torch

import q4_reference as ref
from conftest import pkg

BF16, U8, I32, I64 = torch.bfloat16, torch.uint8, torch.int32, torch.int64


@pytest.fixture(scope='module')
def lib():
    pkg('build').build()
    return pkg('_lib').load()


@pytest.fixture(scope='module')
def q4(lib):
    return pkg('q4')


# ------------------------------------------------------------------------------------ the format
def test_reference_e4m3_is_the_types():
    b = torch.arange(127, dtype=U8)
    np.testing.assert_array_equal(b.view(torch.float8_e4m3fn).float().numpy(), ref.E4M3)
    x = torch.rand(4096, dtype=torch.float32) * 2.0 ** torch.randint(-12, 9, (4096,))
    np.testing.assert_array_equal(x.clamp(max=448).to(torch.float8_e4m3fn).view(U8).numpy(), ref.e4m3_byte(x.numpy()))


@pytest.mark.parametrize('W', [256, 512, 1024])
def test_reference_rows_round_trip_their_bytes(W):
    rng = np.random.default_rng(W)
    cache = np.zeros((3, 1, 32, 17 * W // 16), dtype=np.uint8)
    k, v = rng.standard_normal((2, W))
    ref.put_row(cache, W, 32, 53, k, v, 0.5, 2.0)
    kk, vv = ref.unpack_cache(cache, W)
    np.testing.assert_array_equal(kk[1, 21] * 0.5, ref.stored(k, 0.5))
    np.testing.assert_array_equal(vv[1, 21] * 2.0, ref.stored(v, 2.0))
    assert (kk[1, :21] == 0).all() and (kk[0] == 0).all() and (vv[2] == 0).all()


def test_sizes_and_scales(q4):
    assert [q4.row_bytes(w) for w in (256, 512, 1024)] == [272, 544, 1088]
    assert q4.weight_tiles(1, 32) == (1, 1, 1088) and q4.weight_tiles(33, 2048) == (3, 16, 1088)
    for amax in (1e-6, 0.3, 1.0, 7 * 448, 7 * 448 * 1.001, 1e5):
        ts = q4.tensor_scale(amax)
        assert math.log2(ts).is_integer() and amax / (7 * ts) <= 448 < 2 * amax / (7 * ts) * 1.0000001
    assert q4.tensor_scale(0.0) == 1.0
    cache = q4.new_cache(3, 48, 256, device='cpu')
    assert cache.shape == (3, 1, 48, 272) and cache.dtype == U8 and not cache.any() and q4.cache_width(cache) == 256
    for bad in ((3, 16, 384), (3, 8, 256), (3, 24, 256)):
        with pytest.raises(ValueError, match='4-bit latent cache'):
            q4.new_cache(*bad, device='cpu')


def test_tensor_scale_at_its_ends(q4):
    """Never below fp32's smallest normal number, which is the least a row can be quantised with."""
    for amax in (5e-324, 1e-40, 1e-38, 3136 * 2.0 ** -126):
        assert q4.tensor_scale(amax) == 2.0 ** -126
    assert q4.tensor_scale(3136 * 2.0 ** -126 * 1.001) == 2.0 ** -125
    for amax in (float('nan'), float('inf')):
        with pytest.raises(ValueError, match='finite'):
            q4.tensor_scale(amax)


def test_geometry_check_takes_4_bit_caches(q4):
    geo = pkg('geometry')
    rec = geo.check_latent_caches({512: q4.new_cache(5, 48, 512, 'cpu'), 256: torch.zeros(5, 1, 16, 512, dtype=BF16)})
    assert rec['caches'][512] == [[5, 1, 48, 544], [48 * 544, 48 * 544, 544, 1], 'torch.uint8']
    with pytest.raises(RuntimeError, match='unexpected 4-bit'):
        geo.check_latent_caches({512: q4.new_cache(5, 16, 256, 'cpu')})
    with pytest.raises(RuntimeError, match='unexpected 4-bit'):
        geo.check_latent_caches({512: torch.zeros(5, 1, 8, 544, dtype=U8)})
    with pytest.raises(RuntimeError, match='no instance'):
        geo.check_latent_caches({128: torch.zeros(5, 1, 16, 136, dtype=U8)})
    with pytest.raises(RuntimeError, match='contiguous'):
        geo.check_latent_caches({512: torch.zeros(5, 1, 16, 600, dtype=U8)[..., :544]})


# ------------------------------------------------------------------------------------ refusals of the module
def history_args(**kw):
    a = dict(q_lat=torch.zeros(2, 16, 512, dtype=BF16), cache=torch.zeros(4, 1, 16, 544, dtype=U8),
             block_table=torch.zeros(2, 3, dtype=I32), ctx=torch.zeros(2, dtype=I32), scale=1.0, num_kv_splits=2,
             workspace=pkg('s6_ops').S6Workspace(16, 512, 4))
    a.update(kw)
    return a


@pytest.mark.parametrize('kw,match', [
    (dict(), 'CUDA'),
    (dict(q_lat=torch.zeros(2, 16, 512)), 'q_lat must be bf16'),
    (dict(q_lat=torch.zeros(2, 512, dtype=BF16)), 'q_lat must be bf16'),
    (dict(q_lat=torch.zeros(2, 512, 16, dtype=BF16).transpose(1, 2)), 'unit last-dim'),
    (dict(cache=torch.zeros(4, 1, 16, 272, dtype=U8)), 'width 512 must be uint8'),
    (dict(cache=torch.zeros(4, 1, 16, 544, dtype=torch.int8)), 'width 512 must be uint8'),
    (dict(cache=torch.zeros(4, 16, 544, dtype=U8)), 'width 512 must be uint8'),
    (dict(cache=torch.zeros(4, 1, 16, 1088, dtype=U8)[..., :544]), 'contiguous'),
    (dict(block_table=torch.zeros(2, 3, dtype=I64)), 'int32'),
    (dict(block_table=torch.zeros(1, 3, dtype=I32)), 'row per token'),
    (dict(block_table=torch.zeros(3, 2, dtype=I32).t()), 'unit last-dim'),
    (dict(ctx=torch.zeros(2, dtype=I64)), 'ctx must be int32'),
    (dict(ctx=torch.zeros(3, dtype=I32)), 'ctx must be int32'),
    (dict(empty=torch.zeros(3, dtype=torch.bool)), 'empty must be'),
    (dict(error_flag=torch.zeros(1, dtype=I64)), 'error_flag must be int32'),
    (dict(error_flag=torch.zeros(0, dtype=I32)), 'error_flag must be int32'),
])
def test_history_refusals(q4, kw, match):
    args = history_args(**kw)
    with pytest.raises(ValueError, match=match):
        q4.history_attention(**args)
    assert args['workspace'].buffer is None      # a refused call leaves the workspace for its first use


def commit_args(**kw):
    a = dict(row=torch.zeros(3, 1024, dtype=BF16), positions=torch.zeros(3, dtype=I64),
             table=torch.zeros(64, 512, dtype=BF16), cache=torch.zeros(4, 1, 16, 544, dtype=U8),
             block_table=torch.zeros(2, 3, dtype=I32), query_start_loc=torch.tensor([0, 1, 3], dtype=I32))
    a.update(kw)
    return a


@pytest.mark.parametrize('kw,match', [
    (dict(), 'CUDA'),
    (dict(row=torch.zeros(3, 1024)), 'row must be bf16'),
    (dict(row=torch.zeros(3, 2048, dtype=BF16)[:, ::2]), 'row must be bf16'),
    (dict(row=torch.zeros(3, 512, dtype=BF16)), 'width 256 must be uint8'),
    (dict(positions=torch.zeros(3, dtype=I32)), 'positions must be int64'),
    (dict(positions=torch.zeros(2, dtype=I64)), 'positions must be int64'),
    (dict(table=torch.zeros(64, 256, dtype=BF16)), 'table must be bf16'),
    (dict(table=torch.zeros(64, 512)), 'table must be bf16'),
    (dict(block_table=torch.zeros(1, 3, dtype=I32)), 'block_table'),
    (dict(query_start_loc=torch.zeros(3, dtype=I64)), 'query_start_loc int32'),
])
def test_commit_refusals(q4, kw, match):
    with pytest.raises(ValueError, match=match):
        q4.commit_rows(**commit_args(**kw))


def test_commit_refuses_rows_of_an_odd_width(q4):
    """A column more than K and V have is no row of this cache, though half of it rounds to its width."""
    with pytest.raises(ValueError, match='row must be bf16'):
        q4.commit_rows(**commit_args(row=torch.zeros(3, 1032, dtype=BF16)[:, :1025]))


def test_gather_refusals(q4):
    cache = q4.new_cache(4, 16, 256, 'cpu')
    blocks, slots = torch.zeros(2, dtype=I32), torch.zeros(5, dtype=I64)
    with pytest.raises(ValueError, match='CUDA'):
        q4.gather_rows(cache, blocks, 20)
    with pytest.raises(IndexError, match='does not cover'):
        q4.gather_rows(cache, blocks, 33)
    with pytest.raises(IndexError, match='does not cover'):
        q4.gather_rows(cache, blocks, -1)
    with pytest.raises(ValueError, match='blocks must be int32'):
        q4.gather_rows(cache, blocks.long(), 20)
    with pytest.raises(ValueError, match='slots int64'):
        q4.gather_slots(cache, slots.int())
    with pytest.raises(ValueError, match='out must be bf16'):
        q4.gather_slots(cache, slots, out=torch.zeros(5, 512))
    with pytest.raises(ValueError, match='out must be bf16'):
        q4.gather_slots(cache, slots, out=torch.zeros(4, 512, dtype=BF16))
    with pytest.raises(ValueError, match='4-bit latent cache'):
        q4.gather_slots(cache[:, 0], slots)
    with pytest.raises(ValueError, match='error_flag must be int32'):
        q4.gather_slots(cache, slots, error_flag=torch.zeros(4, dtype=U8))


def test_linear_refusals(q4):
    x, w = torch.zeros(3, 160, dtype=BF16), torch.zeros(2, 2, 1088, dtype=U8)
    with pytest.raises(ValueError, match='CUDA'):
        q4.linear(x, w, 20, 1.0)
    for bad in (w[:1], w[:, :1], w.int(), w.transpose(0, 1)):
        with pytest.raises(ValueError, match='packed must be contiguous uint8'):
            q4.linear(x, bad if bad.shape != w.shape or bad.dtype != U8 else torch.zeros(2, 2, 2176, dtype=U8)[..., ::2],
                      20, 1.0)
    with pytest.raises(ValueError, match='x must be bf16'):
        q4.linear(x.float(), w, 20, 1.0)
    with pytest.raises(ValueError, match='x must be bf16'):
        q4.linear(x[None], w, 20, 1.0)
    for bad in (torch.zeros(3, 21, dtype=BF16), torch.zeros(2, 20, dtype=BF16), torch.zeros(3, 20),
                torch.zeros(20, 3, dtype=BF16).t()):
        with pytest.raises(ValueError, match='residual and out'):
            q4.linear(x, w, 20, 1.0, residual=bad)
        with pytest.raises(ValueError, match='residual and out'):
            q4.linear(x, w, 20, 1.0, out=bad)
    for shape in ((20, 48), (20, 0), (0, 64)):
        with pytest.raises(ValueError, match='multiple of 32'):
            q4.quantize_weight(torch.zeros(shape, dtype=BF16))
    with pytest.raises(ValueError, match='weight must be bf16'):
        q4.quantize_weight(torch.zeros(16, 64))
    with pytest.raises(ValueError, match='CUDA'):
        q4.quantize_weight(torch.zeros(16, 64, dtype=BF16))


def test_linear_refuses_more_tokens_than_its_grid_holds(q4, lib):
    """Above 65535 tiles of 256, and where the count would not fit the entry's 32 bits."""
    w = torch.zeros(1, 1, 1088, dtype=U8)
    for T in (65535 * 256 + 1, 2 ** 31 + 5, 2 ** 32 + 3):
        with pytest.raises(ValueError, match='at most 16776960 tokens'):
            q4.linear(torch.zeros(1, 32, dtype=BF16).expand(T, 32), w, 16, 1.0)
    base = dict(x=A16, st=2048, w=A16, T=65535 * 256 + 1, N=64, K=2048, scale=1.0, res=None, r_st=0, out=A16, o_st=64,
                stream=None)
    refused(lib, 'hla_s6_linear_q4', base, [(dict(), 'at most 16776960 tokens')])


def test_linear_takes_an_error_word(q4, lib):
    """The kernels' bounded waits have somewhere to report to: ``linear``, ``Weight.linear`` and the C entry behind them."""
    x, w = torch.zeros(3, 160, dtype=BF16), torch.zeros(2, 2, 1088, dtype=U8)
    for bad in (torch.zeros(1, dtype=I64), torch.zeros(0, dtype=I32)):
        with pytest.raises(ValueError, match='error_flag must be int32'):
            q4.linear(x, w, 20, 1.0, error_flag=bad)
        with pytest.raises(ValueError, match='error_flag must be int32'):
            q4.Weight(w, 20, 1.0).linear(x, error_flag=bad)
    with pytest.raises(ValueError, match='CUDA'):
        q4.linear(x, w, 20, 1.0, error_flag=torch.zeros(1, dtype=I32))
    base = dict(x=A16, st=2048, w=A16, T=3, N=64, K=2048, scale=1.0, res=None, r_st=0, out=A16, o_st=64, err=A16,
                stream=None)
    refused(lib, 'hla_s6_linear_q4_checked', base, [(dict(T=-1), 'linear'), (dict(o_st=63), 'linear')])


def test_packed_writers_move_with_their_module(q4):
    """``.to`` of a layer, and of what holds it, takes the packed copies along; their bytes keep their type."""
    lat = pkg('latent')
    layer = lat.LatentLayer(64, 2, 128, 3, 256, 256, 256)
    shapes = [(512, 64)] * 3
    layer.packed_writers = [q4.Weight(torch.zeros(q4.weight_tiles(*s), dtype=U8), s[0], 0.5) for s in shapes]
    torch.nn.ModuleList([layer]).to('meta', BF16)
    assert layer.cand1.weight.device.type == 'meta' and layer.cand1.weight.dtype is BF16
    assert len(layer.packed_writers) == 3
    for w, s in zip(layer.packed_writers, shapes):
        assert w.packed.device.type == 'meta' and w.packed.dtype is U8 and w.packed.shape == q4.weight_tiles(*s)
        assert w.out_features == s[0] and w.scale == 0.5
    assert not any('packed' in name for name in layer.state_dict())


def test_callers_refuse_mixed_and_misnamed_caches(q4):
    ce, oa = pkg('cache_export'), pkg('ouro_attention')
    four, two = q4.new_cache(4, 16, 512, 'cpu'), torch.zeros(4, 1, 16, 512, dtype=BF16)
    with pytest.raises(ValueError, match='or 4-bit ones'):
        ce.export_rows([four], [two], [0], [0], 5, 16)
    assert oa.PagedCaches(four, two, None, [], None).main_scale == (1.0, 1.0)


# ------------------------------------------------------------------------------------ refusals of the C entries
# A pointer that is never followed: every call below is refused on the host.
A16, A8 = ctypes.c_void_p(1 << 12), ctypes.c_void_p((1 << 12) + 8)


def refused(lib, name, base, cases):
    _lib = pkg('_lib')
    fn = getattr(lib, name)
    for change, text in cases:
        args = dict(base)
        for key in change:
            assert key in args, key
        args.update(change)
        assert fn(*args.values()) == _lib.EINVAL, (name, change)
        assert text in lib.hla_s6_last_error().decode(), (name, change, lib.hla_s6_last_error())


def test_history_entry_refusals(lib):
    base = dict(q=A16, q_st=8192, q_sh=512, cache=A16, nb=4, sb=16 * 544, bt=A16, bt_st=3, cols=3, ctx=A16, empty=None,
                T=2, H=16, W=512, page=16, scale=1.0, splits=2, ws=A16, floats=1 << 20, ks=1.0, vs=1.0, out=A16,
                o_st=8192, o_sh=512, lse=A16, err=None, stream=None)
    nan, inf = float('nan'), float('inf')
    cases = [(dict(H=0), 'heads'), (dict(H=17), 'heads'), (dict(T=-1), 'heads'), (dict(splits=0), 'num_kv_splits'),
             (dict(W=384), 'width'), (dict(W=128), 'width'), (dict(page=8), 'page'), (dict(page=24), 'page'),
             (dict(q=A8), '16-byte'), (dict(q_st=8196), '16-byte'), (dict(q_sh=516), '16-byte'), (dict(cache=A8), 'base'),
             (dict(sb=16 * 544 + 8), 'stride'), (dict(sb=16 * 544 - 16), 'holds a page'), (dict(nb=0), 'base'),
             (dict(ws=A8), 'workspace')]
    cases += [(dict([(k, x)]), 'tensor scales') for k in ('ks', 'vs') for x in (0.0, -1.0, nan, inf)]
    refused(lib, 'hla_s6_history_attention_q4', base, cases)
    for key in ('empty', 'out', 'o_st', 'o_sh', 'lse', 'err', 'stream'):
        base.pop(key)
    base.update(err=None, flags=0, stream=None)
    refused(lib, 'hla_s6_history_partials_q4', base, cases + [(dict(flags=2), 'flags')])
    base['floats'] = 2 * 16 * 2 * 513 - 1
    assert lib.hla_s6_history_partials_q4(*base.values()) == pkg('_lib').EOVERFLOW


def test_rows_entry_refusals(lib):
    base = dict(row=A16, st=1024, W=512, pos=A16, table=A16, tab_st=512, max_pos=64, cache=A16, nb=4, sb=16 * 544,
                page=16, bt=A16, bt_st=3, cols=3, qsl=A16, R=2, T=3, ks=1.0, vs=1.0, slots=None, stream=None)
    shared = [(dict(W=384), 'width'), (dict(page=24), 'page'), (dict(cache=A8), '16-byte'), (dict(sb=544), 'holds a page'),
              (dict(ks=0.0), 'scales'), (dict(vs=float('nan')), 'scales')]
    refused(lib, 'hla_s6_commit_rows_q4', base, shared + [
        (dict(T=-1), 'commit rows'), (dict(R=0), 'commit rows'), (dict(max_pos=0), 'commit rows'),
        (dict(row=A8), 'commit rows'), (dict(st=1028), 'commit rows'), (dict(tab_st=500), 'commit rows'),
        (dict(table=A8), 'commit rows'), (dict(cols=-1), 'commit rows'), (dict(cols=1 << 28), '2^31')])
    base = dict(cache=A16, nb=4, sb=16 * 544, W=512, page=16, blocks=A16, slots=None, n=20, ks=1.0, vs=1.0, out=A16,
                o_st=1024, err=None, stream=None)
    refused(lib, 'hla_s6_gather_rows_q4', base, shared + [
        (dict(slots=A16), 'gather'), (dict(blocks=None), 'gather'), (dict(n=-1), 'gather'), (dict(n=1 << 31), 'gather'),
        (dict(out=A8), 'gather'), (dict(o_st=1028), 'gather'), (dict(o_st=1016), 'gather')])


def test_entries_that_quantise_refuse_scales_below_the_normal_numbers(lib):
    base = dict(row=A16, st=1024, W=512, pos=A16, table=A16, tab_st=512, max_pos=64, cache=A16, nb=4, sb=16 * 544,
                page=16, bt=A16, bt_st=3, cols=3, qsl=A16, R=2, T=3, ks=1.0, vs=1.0, slots=None, stream=None)
    refused(lib, 'hla_s6_commit_rows_q4', base, [(dict(ks=2.0 ** -127), '2^-126'), (dict(vs=1e-45), '2^-126')])
    base = dict(w=A16, st=64, N=16, K=64, scale=2.0 ** -130, packed=A16, stream=None)
    refused(lib, 'hla_s6_quantize_weight_q4', base, [(dict(), '2^-126')])


def test_linear_entry_refusals(lib):
    base = dict(x=A16, st=2048, w=A16, T=3, N=64, K=2048, scale=1.0, res=None, r_st=0, out=A16, o_st=64, stream=None)
    refused(lib, 'hla_s6_linear_q4', base, [
        (dict(T=-1), 'linear'), (dict(N=0), 'linear'), (dict(K=0), 'linear'), (dict(K=2040), 'linear'),
        (dict(w=A8), 'linear'), (dict(o_st=63), 'linear'), (dict(scale=0.0), 'linear'),
        (dict(scale=float('inf')), 'linear')])
    base = dict(w=A16, st=64, N=16, K=64, scale=1.0, packed=A16, stream=None)
    refused(lib, 'hla_s6_quantize_weight_q4', base, [
        (dict(N=0), 'weight'), (dict(K=48), 'weight'), (dict(w=A8), 'weight'), (dict(st=60), 'weight'),
        (dict(packed=A8), 'weight'), (dict(scale=0.0), 'weight'), (dict(scale=float('nan')), 'weight')])


def test_calls_without_tokens_do_nothing(lib):
    """No token, no launch: OK without a GPU."""
    assert lib.hla_s6_commit_rows_q4(A16, 1024, 512, A16, A16, 512, 64, A16, 4, 16 * 544, 16, A16, 3, 3, A16, 2, 0, 1.0,
                                     1.0, None, None) == 0
    assert lib.hla_s6_linear_q4(A16, 2048, A16, 0, 64, 2048, 1.0, None, 0, A16, 64, None) == 0
    assert lib.hla_s6_gather_rows_q4(A16, 4, 16 * 544, 512, 16, A16, None, 0, 1.0, 1.0, A16, 1024, None, None) == 0
