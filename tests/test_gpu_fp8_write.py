"""The quantising slot write of the 8-bit cache against its definition in 64 bits.  Codes and scales
are compared bit for bit: with power-of-two scales x / s is exact and there is one rounding, to
nearest even, on both sides."""
import math

import pytest
import torch

from tests.fp8_cache import E4M3, as_values, deal_pages, empty_pool, orc, random_pool

pytestmark = pytest.mark.gpu


def _write(key, value, kc, vc, ks, vs, slots):
    """The call on GPU copies; returns the four tensors back on the CPU."""
    from auto_infer_b200 import ops
    dev = [x.cuda() for x in (kc, vc, ks, vs)]
    ops.reshape_and_cache_fp8(key.cuda(), value.cuda(), *dev, torch.as_tensor(slots, dtype=torch.int32).cuda())
    return [x.cpu() for x in dev]


def _check(key, value, kc, vc, ks, vs, slots, status=0):
    from auto_infer_b200 import ops
    got = _write(key, value, kc, vc, ks, vs, slots)
    assert ops.read_status("cuda") == status
    slots = torch.as_tensor(slots).tolist()
    for rows, codes, scale, got_codes, got_scale in ((key, kc, ks, got[0], got[2]), (value, vc, vs, got[1], got[3])):
        want, want_scale = as_values(codes), scale.double()
        orc.write_kv_fp8(rows, want, want_scale, slots)
        assert torch.equal(got_scale.double().nan_to_num(nan=-1), want_scale.nan_to_num(nan=-1))
        assert torch.equal(as_values(got_codes).nan_to_num(nan=1e9), want.nan_to_num(nan=1e9))
    return got


def _rows(g, t, n_kv, spread=1.0):
    x = torch.randn(t, n_kv, 128, generator=g) * torch.exp(spread * torch.randn(t, n_kv, 1, generator=g))
    return x.to(torch.bfloat16)


@pytest.mark.parametrize("bs", [16, 32, 64, 128, 256, 1024])
@pytest.mark.parametrize("n_kv", [1, 2, 3, 8, 9])
def test_chunks_and_decode_rows(bs, n_kv):
    """A mixed step into used pages: decode rows in the middle of pages, chunks that start and end inside one."""
    g = torch.Generator().manual_seed(bs * 10 + n_kv)
    lens, news = [1, bs + 5, 3 * bs, 2 * bs + 7, 4 * bs + 1], [1, 1, 2 * bs + 3, 17, 1]
    blocks, _, slots = deal_pages(g, lens, bs)
    step = torch.cat([s[-n:] for s, n in zip(slots, news)])
    t = len(step)
    kc, ks = random_pool(g, blocks, bs, n_kv)
    vc, vs = random_pool(g, blocks, bs, n_kv)
    _check(_rows(g, t, n_kv), _rows(g, t, n_kv), kc, vc, ks, vs, step)


@pytest.mark.parametrize("t", [1, 2, 31, 33, 700, 2500])
def test_token_counts_into_a_new_pool(t):
    g = torch.Generator().manual_seed(t)
    blocks, _, slots = deal_pages(g, [t], 128)
    kc, ks = empty_pool(blocks, 128, 2)
    vc, vs = empty_pool(blocks, 128, 2)
    _check(_rows(g, t, 2), _rows(g, t, 2), kc, vc, ks, vs, slots[0])


@pytest.mark.parametrize("bs", [16, 128])
def test_any_order_and_repeated_slots(bs):
    """Rows of a page scattered over the call, and slots that occur several times: the last row is kept."""
    g = torch.Generator().manual_seed(5)
    blocks = 9
    slots = torch.randint(0, blocks * bs, (900,), generator=g)
    kc, ks = random_pool(g, blocks, bs, 4)
    vc, vs = random_pool(g, blocks, bs, 4)
    _check(_rows(g, 900, 4), _rows(g, 900, 4), kc, vc, ks, vs, slots)
    same = torch.full((70,), 3 * bs + 7)
    _check(_rows(g, 70, 4), _rows(g, 70, 4), kc, vc, ks, vs, same)


def test_padding_rows_and_slots_outside_the_pool():
    g = torch.Generator().manual_seed(6)
    kc, ks = random_pool(g, 4, 16, 2)
    vc, vs = random_pool(g, 4, 16, 2)
    slots = [-1, 5, 6, -1, 7, -(1 << 31), 40, 41]
    _check(_rows(g, 8, 2), _rows(g, 8, 2), kc, vc, ks, vs, slots)
    from auto_infer_b200 import _lib
    _check(_rows(g, 8, 2), _rows(g, 8, 2), kc, vc, ks, vs, [64, 5, (1 << 31) - 1, 63, 64, 0, -1, 2], _lib.STATUS_BAD_SLOT)
    got = _check(_rows(g, 3, 2), _rows(g, 3, 2), kc, vc, ks, vs, [-1, -1, -1])
    assert torch.equal(got[0].view(torch.uint8), kc.view(torch.uint8)) and torch.equal(got[2], ks)


def test_growth_page_started_anew_and_scales_that_mean_nothing():
    g = torch.Generator().manual_seed(7)
    bs, n_kv = 32, 2
    kc, ks = random_pool(g, 8, bs, n_kv, spread=0)
    vc, vs = random_pool(g, 8, bs, n_kv, spread=0)
    key, value = _rows(g, 8, n_kv, 0), _rows(g, 8, n_kv, 0)
    key[0] *= 1000                                  # page 0 grows by far: its codes underflow step by step
    value[1] *= 3
    key[2], value[2] = 0, 0                         # rows of zeros: the scale stays
    value[3] *= 1e-30                               # a tiny row under a larger scale: all zeros
    for page, s in ((4, 0.0), (5, math.nan), (6, -1.0), (7, math.inf)):
        ks[page] = s
        vs[page] = s
    slots = [0 * bs + 9, 1 * bs + 31, 2 * bs + 1, 3 * bs + 5, 4 * bs + 3, 5 * bs + 3, 6 * bs + 3, 7 * bs + 3]
    _check(key, value, kc, vc, ks, vs, slots)
    _check(key, value, kc, vc, ks, vs, [s // bs * bs for s in slots])      # all pages started anew


def test_scales_that_are_no_powers_of_two():
    """A pool quantised elsewhere: x / s is rounded once in fp32 before the code is; the two roundings
    can differ from one only where x / s lies within 2^-24 of the middle of two codes, which the
    64-bit values of these inputs do not (checked here)."""
    g = torch.Generator().manual_seed(8)
    kc, ks = random_pool(g, 6, 64, 2, spread=0, any_scale=True)
    vc, vs = random_pool(g, 6, 64, 2, spread=0, any_scale=True)
    key, value = _rows(g, 40, 2, 0) * 0.5, _rows(g, 40, 2, 0) * 0.5
    slots = (torch.arange(40) % 6) * 64 + 1 + torch.arange(40) // 6
    for rows, scale in ((key, ks), (value, vs)):
        y = rows.double() / scale.double()[slots // 64][:, :, None]
        assert (y.abs() < 440).all()
        for eps in (-2.0 ** -23, 2.0 ** -23):
            assert torch.equal(orc.e4m3_round(y), orc.e4m3_round(y * (1 + eps)))
    _check(key, value, kc, vc, ks, vs, slots)


def test_extreme_values():
    """bf16 at its ends, infinities and NaN among the rows: NaN codes, scales from the finite elements."""
    kc, ks = empty_pool(3, 16, 1)
    vc, vs = empty_pool(3, 16, 1)
    key = torch.zeros(6, 1, 128)
    big = float(torch.finfo(torch.bfloat16).max)
    key[0, 0, :8] = torch.tensor([big, -big, 1.0, 0.0, -0.0, 2.0 ** -133, big / 448, big / 512])
    key[1, 0, :4] = torch.tensor([math.inf, -math.inf, math.nan, 3.0])
    key[2, 0, :2] = torch.tensor([2.0 ** -133, -2.0 ** -130])      # below the smallest scale's codes
    key[3] = math.nan
    key[4, 0, :4] = torch.tensor([448.0, 449.0, 1.75, 1.7578125])
    key[5, 0, :2] = 1.75
    key = key.to(torch.bfloat16)
    for order in ([0, 1, 2, 3, 4, 5], [5, 4, 3, 2, 1, 0]):
        _check(key, key[order], kc, vc, ks, vs, [0, 1, 16, 17, 32, 33])
        _check(key[1:4], key[order][1:4], kc, vc, ks, vs, [0, 16, 33])


def test_strided_views_other_streams_and_replay():
    """Rows as views of a packed projection, int64 slots, a side stream, and a recorded call replayed
    with other rows and slots."""
    from auto_infer_b200 import ops
    g = torch.Generator().manual_seed(9)
    t, n_kv, bs = 50, 3, 16
    packed = torch.randn(t, 4 + 2 * n_kv * 128 + 12, generator=g).to(torch.bfloat16)
    for lead in (0, 4, 8):                                         # 8 bytes off alignment: copied; 16: used as it is
        key = packed[:, lead:lead + n_kv * 128].unflatten(1, (n_kv, 128))
        value = packed[:, lead + n_kv * 128:lead + 2 * n_kv * 128].unflatten(1, (n_kv, 128))
        kc, ks = random_pool(g, 8, bs, n_kv)
        vc, vs = random_pool(g, 8, bs, n_kv)
        slots = torch.randperm(8 * bs, generator=g)[:t]
        dev = [x.cuda() for x in (kc, vc, ks, vs)]
        pd = packed.cuda()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            ops.reshape_and_cache_fp8(pd[:, lead:lead + n_kv * 128].unflatten(1, (n_kv, 128)),
                                      pd[:, lead + n_kv * 128:lead + 2 * n_kv * 128].unflatten(1, (n_kv, 128)),
                                      *dev, slots.cuda())
        torch.cuda.current_stream().wait_stream(side)
        want, want_scale = as_values(kc), ks.double()
        orc.write_kv_fp8(key, want, want_scale, slots.tolist())
        assert torch.equal(as_values(dev[0]), want) and torch.equal(dev[2].cpu().double(), want_scale)

    kd, vd, sd = torch.zeros(t, n_kv, 128, dtype=torch.bfloat16, device="cuda"), None, None
    vd, sd = torch.zeros_like(kd), torch.full((t,), -1, dtype=torch.int32, device="cuda")
    kc, ks = random_pool(g, 8, bs, n_kv)
    dev = [x.cuda() for x in (kc, kc, ks, ks)]
    ops.reshape_and_cache_fp8(kd, vd, *dev, sd)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.reshape_and_cache_fp8(kd, vd, *dev, sd)
    want, want_scale = as_values(kc), ks.double()
    for _ in range(3):
        rows, slots = _rows(g, t, n_kv), torch.randperm(8 * bs, generator=g)[:t]
        kd.copy_(rows)
        sd.copy_(slots)
        graph.replay()
        orc.write_kv_fp8(rows, want, want_scale, slots.tolist())
        assert torch.equal(as_values(dev[0]), want) and torch.equal(dev[2].cpu().double(), want_scale)
    assert ops.read_status("cuda") == 0


def test_refusals():
    from auto_infer_b200 import ops
    kc, ks = [x.cuda() for x in empty_pool(2, 16, 2)]
    rows, slots = torch.zeros(3, 2, 128, dtype=torch.bfloat16, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    good = dict(key=rows, value=rows, key_cache=kc, value_cache=kc.clone(), key_scale=ks, value_scale=ks.clone(), slot_mapping=slots)
    ops.reshape_and_cache_fp8(**good)
    ops.reshape_and_cache_fp8(**{**good, "key": rows[:0], "value": rows[:0], "slot_mapping": slots[:0]})
    bad = [dict(key=rows.half()), dict(value=rows.float()), dict(key=rows[:2]), dict(key=rows[:, :1]), dict(slot_mapping=slots[:2]),
           dict(key_cache=kc.view(torch.uint8)), dict(value_cache=kc[:1]), dict(key_scale=ks.half()), dict(value_scale=ks[:1]),
           dict(key_cache=kc.transpose(1, 2).contiguous().transpose(1, 2)), dict(key_scale=ks.t().contiguous().t())]
    for change in bad:
        with pytest.raises(ValueError):
            ops.reshape_and_cache_fp8(**{**good, **change})
    with pytest.raises(RuntimeError):
        ops.reshape_and_cache_fp8(**{**good, "key": rows.cpu()})


@pytest.mark.parametrize("old_rows, new_rows", [(1, [50]), (40, [50]), (40, list(range(41, 64)))])
def test_a_scale_that_grows_further_than_a_quotient_can_say(old_rows, new_rows):
    """Rows near the smallest normal numbers, then one near the largest: s_old / s is below what fp32 holds, and the
    old rows become zeros rather than keep codes that now mean something else."""
    g = torch.Generator().manual_seed(9)
    kc, ks = empty_pool(2, 64, 2)
    vc, vs = empty_pool(2, 64, 2)
    tiny = _rows(g, old_rows, 2) * 2.0 ** -124
    first = _check(tiny, tiny, kc, vc, ks, vs, list(range(old_rows)))
    assert first[0].float()[0, :old_rows].abs().sum() > 0
    huge = _rows(g, len(new_rows), 2) * 2.0 ** 100
    got = _check(huge, huge, *first, new_rows)
    assert (as_values(got[0])[0, :old_rows] == 0).all()


def test_slots_of_64_bits_do_not_wrap_into_the_pool():
    from auto_infer_b200 import ops
    g = torch.Generator().manual_seed(10)
    pool = [x.cuda() for x in (*empty_pool(2, 16, 1), *empty_pool(2, 16, 1))]
    kc, ks, vc, vs = pool
    rows = _rows(g, 3, 1).cuda()
    ops.reshape_and_cache_fp8(rows, rows, kc, vc, ks, vs, torch.tensor([2 ** 32 + 5, -2 ** 32 + 6, 7]).cuda())
    assert ops.read_status("cuda") == 1              # the first is past the pool, the second a padding row
    written = kc.view(torch.uint8).view(32, -1).any(-1).nonzero().flatten().tolist()
    assert written == [7]


@pytest.mark.parametrize("n_kv, bs", [(8, 128), (3, 16)])
def test_scales_that_grow_call_after_call(n_kv, bs):
    """Two hundred decode rows, each into a page of its own, larger call after call: every lane of a page's warp goes by the scale
    that was there before one of them replaced it."""
    from auto_infer_b200 import ops
    g = torch.Generator().manual_seed(12)
    pages = 200
    pools = [random_pool(g, pages, bs, n_kv, spread=1.0) for _ in range(2)]
    (kc, ks), (vc, vs) = [[x.cuda() for x in pool] for pool in pools]
    wants = [(as_values(codes), scale.double()) for codes, scale in pools]
    for call in range(8):
        rows = [(_rows(g, pages, n_kv, 0.3).float() * 2.5 ** call).to(torch.bfloat16) for _ in range(2)]
        slots = torch.arange(pages) * bs + 1 + call
        ops.reshape_and_cache_fp8(rows[0].cuda(), rows[1].cuda(), kc, vc, ks, vs, slots.cuda())
        for x, (want, want_scale), codes, scale in zip(rows, wants, (kc, vc), (ks, vs)):
            orc.write_kv_fp8(x, want, want_scale, slots.tolist())
            assert torch.equal(scale.cpu().double(), want_scale), call
            assert torch.equal(as_values(codes), want), call
    assert ops.read_status("cuda") == 0
