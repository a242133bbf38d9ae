"""Wide-query attention over the 8-bit cache against the formula in 64 bits on the same codes.

Tolerance.  Q's two e4m3 terms hold a bf16 element exactly down to 2^-10 of its row's largest, products are
exact and summed in fp32; a weight is rounded once to f16 (2^-11), the output once to bf16 (2^-8):
|err| <= 2^-8 |out| + 2^-11 A, A = sum p |v|, plus 2^-16 A for sums and exp2 and 2^-13 A for what
Q loses below 2^-10 of its row's largest element: at most 2^-18 of the largest per element, against
keys of unit size a score's error stays under 2^-13 for scores of order 1.  Weights below f16's normal
range add what ``smallest_weights`` derives: a row that one key carries, with code 0 in some column, keeps nothing
there of keys whose weights are under 2^-25 of that key's."""
import math

import pytest
import torch

from tests.fp8_cache import attention, deal_pages, random_pool, sink_case, smallest_weights

pytestmark = pytest.mark.gpu


def _case(seed, lens, q_lens, n_q, n_kv, bs, any_scale=False, spread=1.0, q_mul=1.0):
    g = torch.Generator().manual_seed(seed)
    blocks, table, _ = deal_pages(g, lens, bs)
    kc, ks = random_pool(g, blocks, bs, n_kv, any_scale=any_scale, spread=spread)
    vc, vs = random_pool(g, blocks, bs, n_kv, any_scale=any_scale, spread=spread)
    cu = torch.tensor(q_lens).cumsum(0).tolist()
    q = (torch.randn(cu[-1], n_q, 128, generator=g) * q_mul).to(torch.bfloat16)
    return q, kc, vc, ks, vs, table, cu, list(lens), 128 ** -0.5


def _run(q, kc, vc, ks, vs, table, cu, kv, scale, min_rows=0, base=None, capacity=None, **kw):
    from auto_infer_b200 import ops
    plan = ops.PrefillPlan(cu, kv, q.shape[1], kc.shape[2], "cuda", min_rows=min_rows, causal_base=base,
                           capacity_tokens=capacity, capacity_seqs=len(cu) if capacity else None)
    lse = torch.full(q.shape[:2], 7.0, dtype=torch.float32, device="cuda")
    out = ops.paged_prefill_gqa_fp8(q.cuda(), kc.cuda(), vc.cuda(), ks.cuda(), vs.cuda(), table.cuda(), plan, scale,
                                    lse_out=lse, **kw)
    torch.cuda.synchronize()
    assert ops.read_status("cuda") == 0
    return out.cpu(), lse.cpu()


def _check(got, lse, q, kc, vc, ks, vs, table, cu, kv, scale, base=None):
    want, want_lse = attention(q, kc, vc, ks, vs, table, cu, kv, scale, base)
    a = attention(q, kc, vc.float().abs().to(vc.dtype), ks, vs, table, cu, kv, scale, base)[0]
    last = 2.0 ** -8 if got.dtype == torch.bfloat16 else 2.0 ** -24
    tol = last * want.abs() + (2.0 ** -11 + 2.0 ** -13 + 2.0 ** -16) * a * (1 + last)
    tol += smallest_weights(q, kc, vc, ks, vs, table, cu, kv, scale, base) * (1 + last)
    err = (got.double() - want).abs()
    assert (err <= tol).all(), float((err / tol.clamp_min(1e-300)).max())
    empty = want_lse == -math.inf
    assert torch.equal(lse.double() == -math.inf, empty)
    torch.testing.assert_close(lse.double()[~empty], want_lse[~empty], rtol=2.0 ** -16, atol=2.0 ** -14)


@pytest.mark.parametrize("bs", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("n_q, n_kv", [(1, 1), (8, 2), (7, 1), (16, 1), (10, 2)])
def test_geometries(bs, n_q, n_kv):
    lens, q_lens = [130, 300, 17, 257], [130, 45, 17, 1]
    c = _case(bs + n_q, lens, q_lens, n_q, n_kv, bs, any_scale=bs == 32)
    _check(*_run(*c), *c)


@pytest.mark.parametrize("kv, q_len", [(1, 1), (2, 2), (127, 5), (128, 128), (129, 129), (255, 1), (513, 300), (1500, 33)])
def test_lengths(kv, q_len):
    for bs in (16, 128):
        c = _case(kv, [kv], [q_len], 8, 2, bs)
        _check(*_run(*c), *c)


def test_many_items_on_few_ctas():
    """Several items per CTA, short and long, through the work queue and both Q buffers."""
    lens, q_lens = [900, 40, 1, 300, 130, 600, 64, 257, 20], [200, 40, 1, 100, 2, 333, 64, 17, 3]
    for bs in (32, 128):
        c = _case(bs, lens, q_lens, 8, 2, bs)
        first, lse = _run(*c)
        _check(first, lse, *c)
        for ctas in (1, 2, 5):
            got, _ = _run(*c, max_ctas=ctas)
            assert torch.equal(got, first)


def test_rows_without_keys_and_sequences_without_rows():
    lens, q_lens = [5, 0, 60, 0, 200], [40, 3, 0, 0, 33]     # the first 35 rows of sequence 0 see nothing
    for bs in (16, 128):
        c = _case(bs, lens, q_lens, 4, 1, bs)
        fill = torch.full((76, 4, 128), 3.0, dtype=torch.bfloat16, device="cuda")
        _check(*_run(*c, out=fill), *c)
    c = _case(1, [0, 0], [2, 3], 4, 1, 16)
    c = (*c[:5], c[5][:, :0], *c[6:])
    _check(*_run(*c), *c)


def test_narrow_sequences_are_left_alone():
    c = _case(3, [300, 300, 100], [1, 40, 4], 8, 2, 32)
    out = torch.full((45, 8, 128), 5.0, dtype=torch.bfloat16, device="cuda")
    got, lse = _run(*c, min_rows=16, out=out)
    rest = [0, 41, 42, 43, 44]
    assert (got[rest] == 5.0).all() and (lse[rest] == 7.0).all()
    want, want_lse = attention(*c)
    got[rest], lse[rest] = want[rest].to(torch.bfloat16), want_lse[rest].float()
    _check(got, lse, *c)


def test_fp32_output_and_context_parallel_base():
    from auto_infer_b200 import ops
    c = _case(10, [400], [50], 8, 2, 16)
    _check(*_run(*c, out_f32=True), *c)
    want, _ = attention(*c)
    cut = 160
    parts, lses = [], []
    for lo, hi in ((0, cut), (cut, 400)):
        table = c[5][:, lo // 16:hi // 16].contiguous()
        base = [400 - 50 - lo]
        o, l = _run(*c[:5], table, c[6], [hi - lo], c[8], base=base, out_f32=True)
        _check(o, l, *c[:5], table, c[6], [hi - lo], c[8], base)
        parts.append(o.cuda().view(-1, 128))
        lses.append(l.cuda().view(-1))
    out = ops.lse_combine(torch.stack(parts), torch.stack(lses), out_dtype=torch.float32).cpu().view(50, 8, 128)
    a = attention(c[0], c[1], c[2].float().abs().to(c[2].dtype), *c[3:])[0]
    assert ((out.double() - want).abs() <= (2.0 ** -11 + 2.0 ** -12) * a).all()


@pytest.mark.parametrize("bs", [16, 128])
@pytest.mark.parametrize("spread", [0.0, 6.0, 30.0])
def test_page_scales_far_apart(spread, bs):
    g = torch.Generator().manual_seed(int(spread))
    c = list(_case(6, [900, 333], [70, 33], 8, 2, bs, spread=0.0))
    c[4] = torch.exp2((torch.randn(c[4].shape, generator=g) * spread).clamp(-90, 90).round() - 6)
    _check(*_run(*c), *c)
    c[3] = torch.exp2((torch.randn(c[3].shape, generator=g) * min(spread, 2)).round() - 6)
    _check(*_run(*c), *c)


def test_sharp_scores_and_extreme_queries():
    for bs in (16, 128):
        c = list(_case(7, [500], [60], 8, 2, bs, q_mul=40.0))
        want, want_lse = attention(*c)
        got, lse = _run(*c)
        a = attention(c[0], c[1], c[2].float().abs().to(c[2].dtype), *c[3:])[0]
        s = float(want_lse.abs().max())          # errors of a score, and so of a weight, relative to its size
        tol = 2.0 ** -8 * want.abs() + (2.0 ** -11 + 2 * s * 2.0 ** -17) * a * 1.01
        assert ((got.double() - want).abs() <= tol).all()
        torch.testing.assert_close(lse.double(), want_lse, rtol=2.0 ** -16, atol=2.0 ** -14)
        q = c[0].float()
        q[:20] *= 1e-30
        q[20:30] = 0
        q[30:] *= 2.0 ** 100
        c[0] = q.to(torch.bfloat16)
        _check(*[x[:30] for x in _run(*c)], c[0][:30], *c[1:6], [30], [470], c[8])
        c[3] = c[3] * 2.0 ** -106
        _check(*[x[30:] for x in _run(*c)], c[0][30:], *c[1:6], [30], [500], c[8])


def test_codes_past_the_end_and_unused_pages_may_be_anything():
    for bs in (32, 256):
        c = list(_case(8, [20, 177, 300], [20, 30, 100], 8, 2, bs))
        clean, clean_lse = _run(*c)
        used = torch.zeros(c[1].shape[:2], dtype=torch.bool)
        for b, n in enumerate(c[7]):
            pos = torch.arange(n)
            used[c[5][b].long()[pos // bs], pos % bs] = True
        pages = used.any(1)
        for i in (1, 2):
            raw = c[i].view(torch.uint8).clone()
            raw[~used] = 0x7f                        # NaN codes
            c[i] = raw.view(c[i].dtype)
            c[i + 2] = torch.where(pages[:, None], c[i + 2], torch.tensor(math.nan))
        got, lse = _run(*c)
        assert torch.equal(got, clean) and torch.equal(lse, clean_lse)


def test_nan_and_zero_scales_where_they_count():
    for bs in (16, 128):
        c = list(_case(9, [300, 300], [40, 40], 4, 1, bs))
        page = int(c[5][0, 1])
        for i in (3, 4):
            c[i] = c[i].clone()
            c[i][page] = 0.0                         # a page of zero keys / values
            _check(*_run(*c), *c)
        for i in (3, 4):
            d = list(_case(9, [300, 300], [40, 40], 4, 1, bs))
            d[i] = d[i].clone()
            d[i][page] = math.nan
            got, _ = _run(*d)
            assert got[:40].isnan().all() and not got[40:].isnan().any()


def test_strided_query_views_table_slices_streams_and_replay():
    from auto_infer_b200 import ops
    c = _case(11, [300, 145], [60, 33], 8, 2, 16)
    want, _ = _run(*c)
    big = torch.full((5, 40), -7, dtype=torch.int64)
    big[:2, :c[5].shape[1]] = c[5]
    plan = ops.PrefillPlan(c[6], c[7], 8, 2, "cuda")
    dev = [x.cuda() for x in c[1:5]]
    for lead in (0, 4, 8):
        packed = torch.zeros(93, 8 * 128 + 520 + lead, dtype=torch.bfloat16)
        packed[:, lead:lead + 1024] = c[0].reshape(93, -1)
        side = torch.cuda.Stream()
        view = packed.cuda()[:, lead:lead + 1024].unflatten(1, (8, 128))
        table = big.cuda()[:2, :c[5].shape[1]]
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            out = ops.paged_prefill_gqa_fp8(view, *dev, table, plan, c[8])
        side.synchronize()
        assert torch.equal(out.cpu(), want)
    plan = ops.PrefillPlan(c[6], c[7], 8, 2, "cuda", capacity_tokens=93, capacity_seqs=2)
    q, table = c[0].cuda(), c[5].cuda()
    out, graph = torch.empty_like(q), torch.cuda.CUDAGraph()
    ops.paged_prefill_gqa_fp8(q, *dev, table, plan, c[8], out=out)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        ops.paged_prefill_gqa_fp8(q, *dev, table, plan, c[8], out=out)
    for cu, kv in (([40, 93], [200, 145]), ([93, 93], [300, 0]), ([0, 0], [0, 0]), (c[6], c[7])):
        plan.refill(cu, kv)
        out.fill_(3.0)
        graph.replay()
        torch.cuda.synchronize()
        n = cu[-1]
        assert (out[n:] == 3.0).all()
        if n:
            lse = attention(c[0][:n], *c[1:6], cu, kv, c[8])[1].float()
            _check(out[:n].cpu(), lse, c[0][:n], *c[1:6], cu, kv, c[8])
    assert ops.read_status("cuda") == 0


def test_block_ids_outside_the_pool_and_plans_that_outgrow_their_tensors():
    from auto_infer_b200 import _lib, ops
    for bs in (16, 128):
        c = _case(12, [300, 150], [40, 30], 8, 2, bs)
        dev = [x.cuda() for x in c[:6]]
        plan = ops.PrefillPlan(c[6], c[7], 8, 2, "cuda", capacity_tokens=100, capacity_seqs=4)
        good = ops.paged_prefill_gqa_fp8(*dev, plan, c[8])
        table = dev[5].clone()
        table[0, 1] = 1 << 20
        out = ops.paged_prefill_gqa_fp8(*dev[:5], table, plan, c[8])
        assert ops.read_status("cuda") == _lib.STATUS_BAD_BLOCK
        assert torch.equal(out[40:], good[40:]) and out.isfinite().all()
        graph, out = torch.cuda.CUDAGraph(), torch.empty_like(dev[0])
        ops.paged_prefill_gqa_fp8(*dev, plan, c[8], out=out)
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            ops.paged_prefill_gqa_fp8(*dev, plan, c[8], out=out)
        plan.refill([40, 70, 100], [300, 150, 60])           # a third sequence: neither in q nor in the table
        graph.replay()
        assert ops.read_status("cuda") & _lib.STATUS_BAD_LAUNCH
        assert torch.equal(out, good)
        plan.refill([40, 70], [300, 2000])                   # more keys than the table lists
        graph.replay()
        assert ops.read_status("cuda") == _lib.STATUS_BAD_BLOCK
        assert torch.equal(out[:40], good[:40]) and out.isfinite().all()


def test_two_calls_on_two_streams_with_their_own_plans():
    from auto_infer_b200 import ops
    a, b = _case(13, [700, 300], [300, 100], 8, 2, 16), _case(14, [500], [500], 8, 2, 128)
    wants, devs, plans = [], [], []
    for c in (a, b):
        wants.append(_run(*c)[0])
        devs.append([x.cuda() for x in c[:6]])
        plans.append(ops.PrefillPlan(c[6], c[7], 8, 2, "cuda"))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append(ops.paged_prefill_gqa_fp8(*devs[i], plans[i], a[8], max_ctas=70))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o.cpu(), wants[i]) for o in outs[i])


def test_agrees_with_the_decode_form():
    """The same rows through both kernels."""
    from auto_infer_b200 import ops
    c = _case(16, [1000, 333, 64], [2, 2, 1], 8, 2, 64)
    got, lse = _run(*c)
    plan = ops.DecodePlan(c[6], c[7], 8, 2, "cuda")
    other = ops.paged_decode_gqa_fp8(*[x.cuda() for x in c[:6]], plan, c[8]).cpu()
    a = attention(c[0], c[1], c[2].float().abs().to(c[2].dtype), *c[3:])[0]
    assert ((got.double() - other.double()).abs() <= 2.0 ** -7 * got.abs().double() + 2.0 ** -9 * a).all()


def test_refusals():
    from auto_infer_b200 import ops
    c = _case(15, [100, 50], [20, 10], 8, 2, 16)
    q, kc, vc, ks, vs, table = [x.cuda() for x in c[:6]]
    plan = ops.PrefillPlan(c[6], c[7], 8, 2, "cuda")
    good = dict(q=q, key_cache=kc, value_cache=vc, key_scale=ks, value_scale=vs, block_table=table, plan=plan, scale=c[8])
    ops.paged_prefill_gqa_fp8(**good)
    for bad in (dict(q=q.half()), dict(q=q[:, :4]), dict(q=q[:20]), dict(key_cache=kc.float()), dict(value_cache=vc[:1]),
                dict(key_scale=ks[:, :1]), dict(block_table=table[:1]), dict(block_table=table[:, :3]),
                dict(out=torch.empty_like(q).half()), dict(lse_out=torch.empty(30, 4, device="cuda"))):
        with pytest.raises(ValueError):
            ops.paged_prefill_gqa_fp8(**{**good, **bad})
    with pytest.raises(_b200_error()):
        ops.paged_prefill_gqa_fp8(**{**good, "max_ctas": -1})


def _b200_error():
    from auto_infer_b200._lib import B200Error
    return B200Error


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_a_query_that_is_not_finite_spoils_its_own_row_only(bad):
    c = list(_case(31, [300, 40], [45, 40], 8, 2, 32))
    c[0][[3, 60], [1, 7], [0, 127]] = bad
    got, lse = _run(*c)
    spoilt = torch.zeros(got.shape[:2], dtype=torch.bool)
    spoilt[[3, 60], [1, 7]] = True
    assert got[spoilt].isnan().all()
    clean = c[0].clone()
    clean[spoilt] = 0
    want, want_lse = _run(clean, *c[1:])
    assert torch.equal(got[~spoilt], want[~spoilt]) and torch.equal(lse[~spoilt], want_lse[~spoilt])


@pytest.mark.parametrize("rows", [1, 31, 32, 33, 64, 96, 127])
def test_warps_without_rows(rows):
    """Items whose last rows are missing, over an odd and an even number of tiles, before and after full ones on one CTA."""
    lens, q_lens = [700, 128 + rows, 140, 513, rows], [rows, 128, 3, rows, rows]
    for bs in (32, 128):
        c = _case(rows, lens, q_lens, 1, 1, bs)
        first, lse = _run(*c)
        _check(first, lse, *c)
        again, lse2 = _run(*c, max_ctas=1)
        assert torch.equal(first, again) and torch.equal(lse, lse2)


@pytest.mark.parametrize("lens, q_lens, n_q, n_kv", [
    ([9000], [5], 8, 1), ([5000, 300, 2], [7, 40, 2], 8, 2), ([4097, 3000, 0], [130, 9, 3], 4, 1), ([20000], [1], 8, 8),
    ([1500] * 5, [33] * 5, 7, 1), ([130, 6000], [130, 6000 - 5800], 2, 1)])
@pytest.mark.parametrize("bs", [32, 128])
def test_items_cut_along_the_keys(lens, q_lens, n_q, n_kv, bs):
    """Few items over many keys: pieces and their join, with rows that see nothing of the last pieces, into bf16 and
    fp32, the same bits on any number of CTAs, and what an uncut plan gives within the two's tolerances."""
    from auto_infer_b200 import ops
    c = _case(len(lens) + bs, lens, q_lens, n_q, n_kv, bs)
    plan = ops.PrefillPlan(c[6], c[7], n_q, n_kv, "cuda", min_rows=0)
    if max(lens) > 2000:                                 # twelve tiles are not worth a cut
        assert plan.workspace is not None and plan.host[4] > plan.info.num_items and plan.host[7] >= 1
    first, lse = _run(*c)
    _check(first, lse, *c)
    for kw in (dict(max_ctas=3), dict(capacity=c[6][-1] + 4)):
        again, lse2 = _run(*c, **kw)
        assert torch.equal(first, again) and torch.equal(lse, lse2)
    _check(*_run(*c, out_f32=True), *c)
    whole = ops.PrefillPlan(c[6], c[7], n_q, n_kv, "cuda", min_rows=0, split_ctas=0)
    assert whole.workspace is None and not whole.host[4:8].any()
    dev = [x.cuda() for x in c[:6]]
    lse3 = torch.empty_like(lse, device="cuda")
    uncut = ops.paged_prefill_gqa_fp8(*dev, whole, c[8], lse_out=lse3)
    _check(uncut.cpu(), lse3.cpu(), *c)
    kc = (dev[1].float() * dev[3][:, None, :, None]).to(torch.bfloat16)
    vc = (dev[2].float() * dev[4][:, None, :, None]).to(torch.bfloat16)
    wide = [ops.paged_prefill_gqa(dev[0], kc, vc, dev[5], x, c[8]) for x in (plan, whole)]
    assert torch.equal(wide[0], wide[1])                 # the 16-bit kernel does not see the cuts


def test_cut_plans_refilled_and_replayed():
    """One captured launch for steps that are cut, cut otherwise, not cut, and empty."""
    from auto_infer_b200 import ops
    steps = [([9000, 50], [4, 12]), ([700, 6000], [8, 8]), ([60, 60], [8, 8]), ([0, 12000], [1, 15]), ([300, 1], [0, 0])]
    bs, n_q, n_kv, tokens = 64, 8, 1, 16
    cases = [_case(k, lens, q_lens, n_q, n_kv, bs) for k, (lens, q_lens) in enumerate(steps)]
    blocks, width = max(c[1].shape[0] for c in cases), max(c[5].shape[1] for c in cases)
    q = torch.zeros(tokens, n_q, 128, dtype=torch.bfloat16, device="cuda")
    pool = [torch.zeros(blocks, *cases[0][i].shape[1:], dtype=cases[0][i].dtype, device="cuda") for i in (1, 2, 3, 4)]
    table = torch.zeros(2, width, dtype=torch.int32, device="cuda")
    plan = ops.PrefillPlan(cases[0][6], cases[0][7], n_q, n_kv, "cuda", min_rows=0, capacity_tokens=tokens, capacity_seqs=2)
    lse = torch.empty(tokens, n_q, device="cuda")
    ops.paged_prefill_gqa_fp8(q, *pool, table, plan, cases[0][8], lse_out=lse)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.paged_prefill_gqa_fp8(q, *pool, table, plan, cases[0][8], lse_out=lse)
    for c in cases + cases[:2]:
        n = c[6][-1]
        q[:n].copy_(c[0])
        for dst, src in zip(pool, c[1:5]):
            dst[:src.shape[0]].view(torch.uint8).copy_(src.view(torch.uint8))
        table.zero_()
        table[:, :c[5].shape[1]].copy_(c[5])
        out.fill_(3.0)
        lse.fill_(7.0)
        plan.refill(c[6], c[7])
        graph.replay()
        torch.cuda.synchronize()
        assert ops.read_status("cuda") == 0
        if n:
            _check(out[:n].cpu(), lse[:n].cpu(), *c)
        assert (out[n:] == 3.0).all() and (lse[n:] == 7.0).all()


@pytest.mark.parametrize("max_ctas", [1, 2, 3])
def test_warps_that_have_rows_again_in_the_next_item(max_ctas):
    """Items of a few rows between full ones, short and long, odd and even tile counts, one after the other on few CTAs: a
    warp that only kept the barriers going in one item takes part in the next.  Many runs: the order of arrivals varies."""
    from auto_infer_b200 import ops
    q_lens = [3, 128, 1, 128, 33, 128, 64, 2, 128, 5, 97, 128, 1, 1, 128, 40]
    lens = [900, 128, 130, 300, 400, 1000, 64, 513, 257, 5, 200, 700, 1, 260, 129, 380]
    c = _case(17, lens, q_lens, 1, 1, 128)
    first, lse = _run(*c)
    _check(first, lse, *c)
    for split in (0, None):
        plan = ops.PrefillPlan(c[6], c[7], 1, 1, "cuda", min_rows=0, split_ctas=split)
        dev = [x.cuda() for x in c[:6]]
        if split is None:
            first = ops.paged_prefill_gqa_fp8(*dev, plan, c[8]).cpu()
        for _ in range(30):
            got = ops.paged_prefill_gqa_fp8(*dev, plan, c[8], max_ctas=max_ctas)
        assert torch.equal(got.cpu(), first) or split == 0
        _check(got.cpu(), lse, *c)
    assert ops.read_status("cuda") == 0


def test_few_and_many_rows_in_turn_many_times():
    """Pieces and items of 1 to 130 rows follow one another on a CTA in ever new orders: the same bits every time, on any
    number of CTAs, and no wait runs out - also with items that have no tile at all (more queries than keys)."""
    from auto_infer_b200 import ops
    for q_lens, lens, n_q, n_kv, bs in (([33, 64, 130, 1, 100, 1, 3], [129, 129, 6000, 1000, 500, 50, 1000], 8, 8, 256),
                                        ([128, 300, 2, 3, 300, 17, 2], [3000, 300, 6000, 3000, 300, 3000, 128], 32, 8, 16),
                                        ([300, 130, 33, 300, 64, 1], [300, 1, 50, 500, 128, 1], 16, 2, 16),
                                        ([300, 33, 17, 300, 3, 100], [128, 128, 6000, 300, 3, 6000], 32, 8, 128)):
        c = _case(len(q_lens), lens, q_lens, n_q, n_kv, bs)
        dev = [x.cuda() for x in c[:6]]
        plan = ops.PrefillPlan(c[6], c[7], n_q, n_kv, "cuda", min_rows=0)
        whole = ops.PrefillPlan(c[6], c[7], n_q, n_kv, "cuda", min_rows=0, split_ctas=0)
        for x in (plan, whole):
            want = None
            for k in range(120):
                lse = torch.empty(c[6][-1], n_q, device="cuda")
                got = ops.paged_prefill_gqa_fp8(*dev, x, c[8], lse_out=lse, max_ctas=(0, 50, 3, 20, 1)[k % 5], out_f32=True)
                if want is None:
                    want = got, lse
                assert torch.equal(got, want[0]) and torch.equal(lse, want[1]), k
            assert ops.read_status("cuda") == 0
        out, sums = _run(*c)
        _check(out, sums, *c)


@pytest.mark.parametrize("max_ctas", [1, 3, 0])
def test_many_items_without_keys(max_ctas):
    """More queries than keys: item after item that sees nothing comes out as zeros with lse = -inf, the others beside them
    are not disturbed; the kernel over a 16-bit cache has the same queue."""
    from auto_infer_b200 import ops
    c = _case(44, [1, 300, 0, 2], [700, 300, 260, 1], 8, 2, 16)
    dev = [x.cuda() for x in c[:6]]
    plan = ops.PrefillPlan(c[6], c[7], 8, 2, "cuda", min_rows=0)
    want, want_lse = attention(*c)
    empty = want_lse == -math.inf
    kc = (dev[1].float() * dev[3][:, None, :, None]).to(torch.bfloat16)
    vc = (dev[2].float() * dev[4][:, None, :, None]).to(torch.bfloat16)
    for _ in range(20):
        for call in (lambda **kw: ops.paged_prefill_gqa_fp8(*dev, plan, c[8], **kw),
                     lambda **kw: ops.paged_prefill_gqa(dev[0], kc, vc, dev[5], plan, c[8], **kw)):
            lse = torch.full(want_lse.shape, 7.0, device="cuda")
            got = call(lse_out=lse, max_ctas=max_ctas, out=torch.full(want.shape, 3.0, device="cuda"))
            assert torch.equal(lse.cpu() == -math.inf, empty) and (got.cpu()[empty] == 0).all()
            assert (got.cpu().double() - want).abs().max() <= 2.0 ** -5 * want.abs().max()    # bf16 K, V and weights
    assert ops.read_status("cuda") == 0


@pytest.mark.parametrize("bs", [32, 128])
@pytest.mark.parametrize("scale", [-128 ** -0.5, -0.01, -1.0, 0.0])
def test_softmax_scales_that_are_negative_or_zero(scale, bs):
    """The largest score then belongs to the smallest product, and the masked keys stay the smallest: whole items and cut
    ones, and the form for few rows."""
    from auto_infer_b200 import ops
    for lens, q_lens in (([130, 300, 17], [130, 45, 17]), ([5000], [7])):
        c = (*_case(21, lens, q_lens, 8, 2, bs, q_mul=0.5)[:8], scale)
        _check(*_run(*c), *c)
        _check(*_run(*c, out_f32=True), *c)
    c = (*_case(22, [333, 64], [2, 1], 8, 2, bs, q_mul=0.5)[:8], scale)
    plan = ops.DecodePlan(c[6], c[7], 8, 2, "cuda")
    lse = torch.empty(3, 8, device="cuda")
    got = ops.paged_decode_gqa_fp8(*[x.cuda() for x in c[:6]], plan, scale, lse_out=lse)
    _check(got.cpu(), lse.cpu(), *c)


@pytest.mark.parametrize("mass", [0.9, 0.99, 0.999])
@pytest.mark.parametrize("sink_v", [0.0, 0.005])
@pytest.mark.parametrize("n, q_len, bs, split", [(131072, 3, 128, 0), (131072, 3, 128, None), (9000, 20, 16, 0), (9000, 20, 128, 0)])
def test_many_small_weights_beside_a_key_that_carries_the_row(mass, sink_v, n, q_len, bs, split):
    """Tolerance: a row's largest weight is 2^7 at least of the reference that ``smallest_weights`` takes as 1, so what it derives
    for weights below f16's normal range is 2^-7 of it.  O is summed over n / 16 steps of the product in fp32, each
    off by 2^-24 of the sum so far at most; the rest as above."""
    from auto_infer_b200 import ops
    c = sink_case(43, [n], [q_len], 8, bs, mass, sink_v)
    plan = ops.PrefillPlan(c[6], c[7], 8, 1, "cuda", min_rows=0, split_ctas=split)
    lse = torch.empty(q_len, 8, device="cuda")
    got = ops.paged_prefill_gqa_fp8(*[x.cuda() for x in c[:6]], plan, c[8], lse_out=lse, out_f32=True).cpu()
    assert ops.read_status("cuda") == 0
    want, want_lse = attention(*c)
    a = attention(c[0], c[1], c[2].float().abs().to(c[2].dtype), *c[3:])[0]
    tol = (2.0 ** -11 + 2.0 ** -13 + 2.0 ** -16 + n / 16 * 2.0 ** -24) * a + 2.0 ** -7 * smallest_weights(*c)
    err = (got.double() - want).abs()
    assert (err <= tol).all(), float((err / tol).max())
    torch.testing.assert_close(lse.cpu().double(), want_lse, rtol=2.0 ** -16, atol=2.0 ** -14)


def test_a_plan_is_cut_and_has_a_workspace_when_that_is_needed():
    """Neither for the 16-bit kernel; from the first launch over an 8-bit cache on, with room for what the step needs in an
    eager launch and for what any step needs in a recorded one."""
    from auto_infer_b200 import ops
    c = _case(45, [9000, 50], [4, 12], 8, 1, 64)
    dev = [x.cuda() for x in c[:6]]
    kc = (dev[1].float() * dev[3][:, None, :, None]).to(torch.bfloat16)
    vc = (dev[2].float() * dev[4][:, None, :, None]).to(torch.bfloat16)
    want, lse = _run(*c)
    _check(want, lse, *c)
    record = 128 * 129 * 4
    for capacity in (None, 16):
        before = torch.cuda.memory_allocated()
        plan = ops.PrefillPlan(c[6], c[7], 8, 1, "cuda", min_rows=0, capacity_tokens=capacity, capacity_seqs=capacity and 2)
        wide = ops.paged_prefill_gqa(dev[0], kc, vc, dev[5], plan, c[8])
        if capacity:
            plan.refill(c[6], c[7])
            assert torch.equal(ops.paged_prefill_gqa(dev[0], kc, vc, dev[5], plan, c[8]), wide)
        assert not plan.host[4:8].any() and torch.cuda.memory_allocated() - before < record
        for _ in range(2):
            assert torch.equal(ops.paged_prefill_gqa_fp8(*dev, plan, c[8]).cpu(), want)
            assert plan.host[4] > 0 and 2 * record <= plan.workspace.numel() < ops.sm_count() * record
            assert torch.equal(ops.paged_prefill_gqa(dev[0], kc, vc, dev[5], plan, c[8]), wide)
            if capacity:
                plan.refill(c[6], c[7])
                assert plan.host[4] > 0
    asked = ops.PrefillPlan(c[6], c[7], 8, 1, "cuda", min_rows=0, split_ctas=ops.sm_count())
    assert torch.equal(asked.host[:asked.info.plan_ints], plan.host[:plan.info.plan_ints])
    for first in (True, False):                          # the recorded launch is the plan's first over an 8-bit cache
        if first:
            plan = ops.PrefillPlan(c[6], c[7], 8, 1, "cuda", min_rows=0, capacity_tokens=16, capacity_seqs=2)
        graph, out = torch.cuda.CUDAGraph(), torch.empty_like(dev[0])
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            ops.paged_prefill_gqa_fp8(*dev, plan, c[8], out=out)
        assert plan._workspace.numel() >= 2 * ops.sm_count() * record
        graph.replay()
        lse = attention(*c)[1].float()
        _check(out.cpu(), lse, *c)
        held = plan._workspace.data_ptr()
        for _ in range(2):
            plan.refill(c[6], c[7])
            out.fill_(3.0)
            graph.replay()
            assert torch.equal(out.cpu(), want)
            assert torch.equal(ops.paged_prefill_gqa_fp8(*dev, plan, c[8]).cpu(), want) and plan._workspace.data_ptr() == held
    assert ops.read_status("cuda") == 0


@pytest.mark.parametrize("max_ctas", [1, 2, 3])
@pytest.mark.parametrize("split", [0, None])
def test_every_launch_of_items_with_and_without_rows_gives_the_same_bits(split, max_ctas):
    """Output and sums of each of many launches, whole items and cut ones, on few CTAs, where a warp that has no row in one item
    has some in the next: all like the first launch's, and that one right."""
    from auto_infer_b200 import ops
    q_lens = [3, 128, 1, 128, 33, 128, 64, 2, 128, 5, 97, 128, 1, 1, 128, 40]
    lens = [900, 128, 130, 300, 400, 1000, 64, 513, 257, 5, 200, 700, 1, 260, 129, 380]
    for bs in (32, 128):
        c = _case(17, lens, q_lens, 1, 1, bs)
        dev = [x.cuda() for x in c[:6]]
        plan = ops.PrefillPlan(c[6], c[7], 1, 1, "cuda", min_rows=0, split_ctas=split)
        calls = []
        for _ in range(30):
            lse = torch.full((c[6][-1], 1), 7.0, device="cuda")
            out = torch.full_like(dev[0], 3.0)
            ops.paged_prefill_gqa_fp8(*dev, plan, c[8], out=out, lse_out=lse, max_ctas=max_ctas)
            calls.append((out, lse))
        _check(*[x.cpu() for x in calls[0]], *c)
        assert all(torch.equal(out, calls[0][0]) and torch.equal(lse, calls[0][1]) for out, lse in calls)
    assert ops.read_status("cuda") == 0
