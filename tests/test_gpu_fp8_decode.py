"""Decode / verify attention over the 8-bit cache against the formula in 64 bits on the same codes.

Tolerance.  Products of Q (exact in f16) and codes are exact and summed in fp32, the weights are
rounded once to f16 (half a step: 2^-11 relative), the output once to bf16 (2^-8).  A weight's
rounding moves the output by at most 2^-11 sum p |v| / l, so
|err| <= 2^-8 |out| + 2^-11 A + fp32 noise, A = sum p |v|; the noise of sums and exp2 is taken as 2^-16 A.
Weights below f16's normal range add what ``smallest_weights`` derives."""
import math

import pytest
import torch

from tests.fp8_cache import attention, deal_pages, random_pool, sink_case, smallest_weights

pytestmark = pytest.mark.gpu


def _magnitude(q, kc, vc, ks, vs, table, cu, kv, scale, base=None):
    """sum p |v| per output element."""
    return attention(q, kc, vc.float().abs().to(vc.dtype), ks, vs, table, cu, kv, scale, base)[0]


def _run(q, kc, vc, ks, vs, table, cu, kv, scale, num_ctas=None, base=None, capacity=None, **kw):
    from auto_infer_b200 import ops
    plan = ops.DecodePlan(cu, kv, q.shape[1], kc.shape[2], "cuda", num_ctas=num_ctas, causal_base=base,
                          capacity_seqs=capacity)
    lse = torch.full(q.shape[:2], 7.0, dtype=torch.float32, device="cuda")
    out = ops.paged_decode_gqa_fp8(q.cuda(), kc.cuda(), vc.cuda(), ks.cuda(), vs.cuda(), table.cuda(), plan, scale,
                                   lse_out=lse, **kw)
    torch.cuda.synchronize()
    assert ops.read_status("cuda") == 0
    return out.cpu(), lse.cpu()


def _check(got, lse, q, kc, vc, ks, vs, table, cu, kv, scale, base=None):
    want, want_lse = attention(q, kc, vc, ks, vs, table, cu, kv, scale, base)
    a = _magnitude(q, kc, vc, ks, vs, table, cu, kv, scale, base)
    last = 2.0 ** -8 if got.dtype == torch.bfloat16 else 2.0 ** -24
    tol = last * want.abs() + (2.0 ** -11 + 2.0 ** -16) * a * (1 + last)
    tol += smallest_weights(q, kc, vc, ks, vs, table, cu, kv, scale, base) * (1 + last)
    err = (got.double() - want).abs()
    assert (err <= tol).all(), float((err / tol.clamp_min(1e-300)).max())
    empty = want_lse == -math.inf
    assert torch.equal(lse.double() == -math.inf, empty)
    # scores of up to ~30: 128 products summed in fp32 and one factor, 2^-20 relative; the sum's log as much again
    torch.testing.assert_close(lse.double()[~empty], want_lse[~empty], rtol=2.0 ** -18, atol=2.0 ** -16)


def _case(seed, lens, q_lens, n_q, n_kv, bs, any_scale=False, spread=1.0, q_mul=1.0):
    g = torch.Generator().manual_seed(seed)
    blocks, table, _ = deal_pages(g, lens, bs)
    kc, ks = random_pool(g, blocks, bs, n_kv, any_scale=any_scale, spread=spread)
    vc, vs = random_pool(g, blocks, bs, n_kv, any_scale=any_scale, spread=spread)
    cu = torch.tensor(q_lens).cumsum(0).tolist()
    q = (torch.randn(cu[-1], n_q, 128, generator=g) * q_mul).to(torch.bfloat16)
    return q, kc, vc, ks, vs, table, cu, list(lens), 128 ** -0.5


@pytest.mark.parametrize("bs", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("n_q, n_kv", [(1, 1), (16, 8), (6, 2), (7, 1), (32, 2), (10, 2)])
def test_geometries(bs, n_q, n_kv):
    lens = [1, 15, 16, 17, 63, 64, 65, 200, 700]
    c = _case(bs + n_q, lens, [1] * len(lens), n_q, n_kv, bs, any_scale=bs == 32)
    for num_ctas in (None, 3):
        _check(*_run(*c, num_ctas=num_ctas), *c)


@pytest.mark.parametrize("q_len", [1, 2, 3, 4])
def test_verify_rows_and_queries_without_keys(q_len):
    """Several query rows a sequence, a sequence shorter than its query block (its first rows see
    nothing), one without keys, one without queries."""
    lens, q_lens = [q_len, 130, 1, 0, 40, 64], [q_len, q_len, q_len, 1, 0, q_len]
    c = _case(q_len, lens, q_lens, 8, 2, 16)
    _check(*_run(*c, out=torch.full((c[0].shape[0], 8, 128), 3.0, dtype=torch.bfloat16, device="cuda")), *c)
    c = _case(q_len, [0, 0], [1, q_len], 8, 2, 16)
    _check(*_run(*c, out=torch.full((1 + q_len, 8, 128), 3.0, dtype=torch.bfloat16, device="cuda")), *c)
    c = (*c[:5], c[5][:, :0], *c[6:])                # no block at all in the table
    _check(*_run(*c, out=torch.full((1 + q_len, 8, 128), 3.0, dtype=torch.bfloat16, device="cuda")), *c)


def test_wide_sequences_are_left_alone():
    c = _case(3, [300, 300, 100], [1, 40, 2], 8, 2, 32)
    out = torch.full((43, 8, 128), 5.0, dtype=torch.bfloat16, device="cuda")
    got, lse = _run(*c, out=out)
    assert (got[1:41] == 5.0).all() and (lse[1:41] == 7.0).all()
    want, want_lse = attention(*c)
    got[1:41], lse[1:41] = want[1:41].to(torch.bfloat16), want_lse[1:41].float()
    _check(got, lse, *c)


def test_long_context_cut_into_pieces_and_fp32_output():
    c = _case(4, [9000, 20000], [1, 2], 8, 1, 128)
    for num_ctas in (1, 7, 148):
        _check(*_run(*c, num_ctas=num_ctas, out_f32=True), *c)


def test_same_result_every_time():
    from auto_infer_b200 import ops
    c = _case(5, [5000, 3, 777, 4096], [1, 1, 2, 1], 16, 2, 64)
    first, lse = _run(*c)
    plan = ops.DecodePlan(c[6], c[7], 16, 2, "cuda")
    dev = [x.cuda() for x in c[:6]]
    for _ in range(20):
        assert torch.equal(ops.paged_decode_gqa_fp8(*dev, plan, c[8]).cpu(), first)
    _check(first, lse, *c)


@pytest.mark.parametrize("spread", [0.0, 6.0, 30.0])
def test_page_scales_far_apart(spread):
    """Neighbouring pages whose scales differ by many powers of two, for K and for V: the weights are
    taken relative to the largest contribution, not to the largest probability."""
    g = torch.Generator().manual_seed(int(spread))
    c = list(_case(6, [900, 33, 256], [1, 1, 2], 8, 2, 16, spread=0.0))
    c[4] = torch.exp2((torch.randn(c[4].shape, generator=g) * spread).clamp(-90, 90).round() - 6)
    _check(*_run(*c), *c)
    c[3] = torch.exp2((torch.randn(c[3].shape, generator=g) * min(spread, 3)).round() - 6)
    _check(*_run(*c), *c)


def test_sharp_scores_and_extreme_queries():
    """Scores of hundreds (one key takes all), queries near bf16's ends, rows of zeros."""
    c = list(_case(7, [500, 77, 200, 300], [1, 1, 1, 1], 8, 2, 16, q_mul=40.0))
    want, want_lse = attention(*c)
    got, lse = _run(*c)
    a = _magnitude(*c)
    # a score of size s carries an error of about 2^-21 s from its fp32 sum: so do the weights, relatively
    s = float(want_lse.abs().max())
    tol = 2.0 ** -8 * want.abs() + (2.0 ** -11 + 2 * s * 2.0 ** -20) * a * 1.01 + smallest_weights(*c)
    assert ((got.double() - want).abs() <= tol).all()
    torch.testing.assert_close(lse.double(), want_lse, rtol=2.0 ** -18, atol=2.0 ** -16)
    q = c[0].float()
    q[1] *= 1e-30                                    # scores of zero: a plain mean
    q[2] = 0
    q[3, :4] *= 2.0 ** 100
    c[0] = q.to(torch.bfloat16)
    ks = c[3].clone()
    c[3] = ks * 1.0
    c[3][c[5][3].long()] *= 2.0 ** -100              # the fourth sequence's keys as small as its queries are large
    c[0][3, 4:] *= 2.0 ** 100
    _check(*[x[1:] if i < 2 else x for i, x in enumerate(_run(*c))], c[0][1:], *c[1:5], c[5][1:], [1, 2, 3], c[7][1:], c[8])


def test_codes_past_the_end_and_unused_pages_may_be_anything():
    c = list(_case(8, [1, 17, 100], [1, 1, 1], 8, 2, 32))
    clean, _ = _run(*c)
    used = torch.zeros(c[1].shape[:2], dtype=torch.bool)
    for b, n in enumerate(c[7]):
        pos = torch.arange(n)
        used[c[5][b].long()[pos // 32], pos % 32] = True
    pages = used.any(1)
    for i in (1, 2):
        raw = c[i].view(torch.uint8).clone()
        raw[~used] = 0x7f                            # NaN codes
        c[i] = raw.view(c[i].dtype)
        c[i + 2] = torch.where(pages[:, None], c[i + 2], torch.tensor(math.nan))
    got, lse = _run(*c)
    assert torch.equal(got, clean)


def test_nan_and_zero_scales_where_they_count():
    c = list(_case(9, [64, 64], [1, 1], 4, 1, 16))
    page = int(c[5][0, 1])
    c[4] = c[4].clone()
    c[4][page] = 0.0                                 # a page of zero values
    _check(*_run(*c), *c)
    c[2] = c[2].clone()
    raw = c[2].view(torch.uint8)
    raw[page, 3] = 0x7f                              # a NaN in a visible row: NaN for its sequence, and for it alone
    got, _ = _run(*c)
    assert got[0].isnan().all() and not got[1].isnan().any()
    c = list(_case(9, [64, 64], [1, 1], 4, 1, 16))
    c[4][page] = math.nan
    got, _ = _run(*c)
    assert got[0].isnan().all() and not got[1].isnan().any()


def test_context_parallel_base_and_merge():
    """Two slices of one sequence with a shifted causal base, merged by their log-sum-exp."""
    from auto_infer_b200 import ops
    c = _case(10, [400], [2], 8, 2, 16)
    want, want_lse = attention(*c)
    cut = 160
    parts, lses = [], []
    for lo, hi in ((0, cut), (cut, 400)):
        table = c[5][:, lo // 16:hi // 16].contiguous()
        o, l = _run(*c[:5], table, c[6], [hi - lo], c[8], base=[398 - lo], out_f32=True)
        parts.append(o.cuda().view(16, 128))
        lses.append(l.cuda().view(16))
    out = ops.lse_combine(torch.stack(parts), torch.stack(lses), out_dtype=torch.float32).cpu().view(2, 8, 128)
    a = _magnitude(*c)
    assert ((out.double() - want).abs() <= (2.0 ** -11 + 2.0 ** -15) * a + smallest_weights(*c)).all()


def test_strided_query_views_table_slices_and_streams():
    from auto_infer_b200 import ops
    c = _case(11, [300, 45, 129], [1, 1, 1], 8, 2, 16)
    want, _ = _run(*c)
    big = torch.full((5, 40), -7, dtype=torch.int64)
    big[:3, :c[5].shape[1]] = c[5]
    plan = ops.DecodePlan(c[6], c[7], 8, 2, "cuda")
    dev = [x.cuda() for x in c[1:5]]
    for lead in (0, 2, 8):
        packed = torch.zeros(3, 8 * 128 + 514 + lead, dtype=torch.bfloat16)
        packed[:, lead:lead + 1024] = c[0].reshape(3, -1)
        side = torch.cuda.Stream()
        view = packed.cuda()[:, lead:lead + 1024].unflatten(1, (8, 128))
        table = big.cuda()[:3, :c[5].shape[1]]
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            out = ops.paged_decode_gqa_fp8(view, *dev, table, plan, c[8])
        side.synchronize()
        assert torch.equal(out.cpu(), want)
    assert ops.read_status("cuda") == 0


def test_block_ids_outside_the_pool_and_plans_that_outgrow_their_tensors():
    from auto_infer_b200 import _lib, ops
    c = _case(12, [100, 50], [1, 1], 8, 2, 16)
    dev = [x.cuda() for x in c[:6]]
    plan = ops.DecodePlan(c[6], c[7], 8, 2, "cuda")
    good = ops.paged_decode_gqa_fp8(*dev, plan, c[8])
    table = dev[5].clone()
    table[0, 2] = 1 << 20
    out = ops.paged_decode_gqa_fp8(*dev[:5], table, plan, c[8])
    assert ops.read_status("cuda") == _lib.STATUS_BAD_BLOCK
    assert torch.equal(out[1], good[1]) and out.isfinite().all()
    # a replayable plan refilled, behind the wrapper's checks, for a step larger than the tensors it was recorded with
    plan = ops.DecodePlan(c[6], c[7], 8, 2, "cuda", capacity_seqs=4)
    graph, out = torch.cuda.CUDAGraph(), torch.empty_like(dev[0])
    ops.paged_decode_gqa_fp8(*dev, plan, c[8], out=out)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        ops.paged_decode_gqa_fp8(*dev, plan, c[8], out=out)
    plan.refill([1, 2, 3], [100, 50, 20])
    graph.replay()
    assert ops.read_status("cuda") & _lib.STATUS_BAD_LAUNCH
    torch.testing.assert_close(out.double(), good.double(), rtol=2 ** -7, atol=0.05)   # other pieces, same rows
    plan.refill([1, 2], [100, 1000])
    graph.replay()
    assert ops.read_status("cuda") == _lib.STATUS_BAD_BLOCK
    torch.testing.assert_close(out[0].double(), good[0].double(), rtol=2 ** -7, atol=0.05)
    assert out.isfinite().all()
    plan.refill([1, 2], [60, 50])
    graph.replay()
    want, _ = attention(*c[:7], [60, 50], c[8])
    assert ops.read_status("cuda") == 0
    torch.testing.assert_close(out.cpu().double(), want, rtol=2 ** -7, atol=0.05)


def test_two_calls_on_two_streams_with_their_own_plans():
    from auto_infer_b200 import ops
    a, b = _case(13, [4000, 900], [1, 1], 8, 2, 16), _case(14, [2500, 3000], [2, 1], 8, 2, 64)
    wants, devs, plans = [], [], []
    for c in (a, b):
        wants.append(_run(*c)[0])
        devs.append([x.cuda() for x in c[:6]])
        plans.append(ops.DecodePlan(c[6], c[7], 8, 2, "cuda"))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append(ops.paged_decode_gqa_fp8(*devs[i], plans[i], a[8]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o.cpu(), wants[i]) for o in outs[i])


def test_refusals():
    from auto_infer_b200 import ops
    c = _case(15, [100, 50], [1, 1], 8, 2, 16)
    q, kc, vc, ks, vs, table = [x.cuda() for x in c[:6]]
    plan = ops.DecodePlan(c[6], c[7], 8, 2, "cuda")
    good = dict(q=q, key_cache=kc, value_cache=vc, key_scale=ks, value_scale=vs, block_table=table, plan=plan, scale=c[8])
    ops.paged_decode_gqa_fp8(**good)
    lse = torch.empty(2, 8, device="cuda")
    for bad in (dict(q=q.half()), dict(q=q[:, :4]), dict(q=q[:1]), dict(q=q[:, :, :64]), dict(key_cache=kc.float()),
                dict(value_cache=vc[:1]), dict(key_scale=ks[:, :1]), dict(value_scale=vs.double()),
                dict(block_table=table[:1]), dict(block_table=table[:, :3]), dict(block_table=table[0]),
                dict(out=torch.empty(2, 8, 64, dtype=torch.bfloat16, device="cuda")), dict(out=torch.empty_like(q).half()),
                dict(out=torch.empty(2, 16, 128, dtype=torch.bfloat16, device="cuda")[:, ::2]),
                dict(lse_out=lse.double()), dict(lse_out=lse[:1])):
        with pytest.raises(ValueError):
            ops.paged_decode_gqa_fp8(**{**good, **bad})
    with pytest.raises(RuntimeError):
        ops.paged_decode_gqa_fp8(**{**good, "block_table": table.cpu()})
    empty = ops.DecodePlan([], [], 8, 2, "cuda")
    assert ops.paged_decode_gqa_fp8(**{**good, "plan": empty, "q": q[:0], "block_table": table[:0]}).shape == (0, 8, 128)


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("num_ctas", [1, 148])
def test_a_query_that_is_not_finite_spoils_its_own_row_only(bad, num_ctas):
    """Also where it makes every score -inf, and where its keys are cut across CTAs; a NaN key is no empty row either."""
    c = list(_case(31, [3000, 40], [2, 1], 8, 2, 32))
    c[0][[1, 2], [5, 0], [0, 127]] = bad
    spoilt = torch.zeros(c[0].shape[:2], dtype=torch.bool)
    spoilt[[1, 2], [5, 0]] = True
    c[1][:, :, :, 0] = torch.tensor(1.0).to(c[1].dtype)      # the scores against the bad element all have one sign
    got, lse = _run(*c, num_ctas=num_ctas)
    assert got[spoilt].isnan().all() and lse[spoilt].isnan().all()
    clean = c[0].clone()
    clean[spoilt] = 0
    want, want_lse = _run(clean, *c[1:], num_ctas=num_ctas)
    assert torch.equal(got[~spoilt], want[~spoilt]) and torch.equal(lse[~spoilt], want_lse[~spoilt])


def test_plans_of_another_kind_are_refused():
    from auto_infer_b200 import ops
    c = _case(32, [100, 50], [1, 30], 8, 2, 16)
    dev = [x.cuda() for x in c[:6]]
    decode = ops.DecodePlan(c[6], c[7], 8, 2, "cuda", capacity_seqs=2)
    prefill = ops.PrefillPlan(c[6], c[7], 8, 2, "cuda", capacity_tokens=31, capacity_seqs=2)
    latent = ops.MlaDecodePlan([1], [50], 2, "cuda")
    for call, plans in ((ops.paged_decode_gqa_fp8, (prefill, latent)), (ops.paged_prefill_gqa_fp8, (decode, latent))):
        for plan in plans:
            with pytest.raises(ValueError, match="the plan must be"):
                call(*dev, plan, c[8])


@pytest.mark.parametrize("mass", [0.9, 0.99, 0.999])
@pytest.mark.parametrize("sink_v", [0.0, 0.005])
@pytest.mark.parametrize("n, q_len, num_ctas", [(131072, 1, 1), (131072, 2, 148), (9000, 1, 2)])
def test_many_small_weights_beside_a_key_that_carries_the_row(mass, sink_v, n, q_len, num_ctas):
    """Tolerance: the largest P of a row is 2^15 at least of the reference ``smallest_weights`` takes as 1, so what it derives for
    weights below f16's normal range is 2^-15 of it.  O is summed over n / 16 steps of the product in fp32, each off by
    2^-24 of the sum so far at most; the rest as above."""
    c = sink_case(41, [n], [q_len], 8, 16 if n < 10000 else 128, mass, sink_v)
    got, lse = _run(*c, num_ctas=num_ctas, out_f32=True)
    want, want_lse = attention(*c)
    a = _magnitude(*c)
    tol = (2.0 ** -11 + 2.0 ** -16 + n / 16 * 2.0 ** -24) * a + 2.0 ** -15 * smallest_weights(*c)
    err = (got.double() - want).abs()
    assert (err <= tol).all(), float((err / tol).max())
    torch.testing.assert_close(lse.double(), want_lse, rtol=2.0 ** -18, atol=2.0 ** -16)


@pytest.mark.parametrize("share", [0.0, 0.3, 0.5, 0.9])
def test_a_workspace_that_is_too_small_spoils_its_own_launch_only(share):
    """The replayable launch cannot know what the plan needs: it says so in the status word, puts the counters of the cut pairs
    back to zero all the same, and the plan gives the right rows with the workspace it asks for."""
    from auto_infer_b200 import _lib, ops
    c = _case(46, [9000, 5000, 40], [1, 2, 1], 8, 2, 64)
    q, kc, vc, ks, vs, table = [x.cuda() for x in c[:6]]
    plan = ops.DecodePlan(c[6], c[7], 8, 2, "cuda", capacity_seqs=3)
    want = ops.paged_decode_gqa_fp8(q, kc, vc, ks, vs, table, plan, c[8])
    record = (16 * 128 + 16) * 4
    assert plan.info.num_partials > 8
    small = int(plan.info.num_partials * share) * record
    lib, out, lse = _lib.load(), torch.empty_like(q), torch.empty(4, 8, device="cuda")
    for nbytes, status in ((small, _lib.STATUS_BAD_LAUNCH), (plan.workspace.numel(), 0), (small, _lib.STATUS_BAD_LAUNCH),
                           (small, _lib.STATUS_BAD_LAUNCH), (plan.workspace.numel(), 0), (plan.workspace.numel(), 0)):
        out.fill_(3.0)
        plan.workspace.view(torch.float32).fill_(math.nan)   # no record of an earlier launch is left
        assert lib.b200_paged_decode_gqa_fp8(
            q.data_ptr(), q.stride(0), kc.data_ptr(), vc.data_ptr(), ks.data_ptr(), vs.data_ptr(), kc.shape[0], 64,
            table.data_ptr(), table.stride(0), *table.shape, plan.dev.data_ptr(), None, plan.num_ctas, 4, 8, 2, 128, c[8],
            plan.workspace.data_ptr(), nbytes, out.data_ptr(), 0, lse.data_ptr(), ops.status_word("cuda").data_ptr(),
            torch.cuda.current_stream().cuda_stream) == 0
        assert ops.read_status("cuda") == status
        pairs, at = int(plan.host[4]), int(plan.host[7])
        assert pairs == 4 and not plan.dev[at:at + 8 * pairs].view(pairs, 8)[:, 5].any()
        if not status:
            assert torch.equal(out, want)
    _check(out.cpu(), lse.cpu(), *c)
