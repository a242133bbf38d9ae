"""The GQA backend over an 8-bit cache: slot write and attention together, step after step, as the engine drives them.

After every step the caches equal the write's definition bit for bit, and the output is compared with the formula
in 64 bits on those codes.  Tolerance: a step may mix both attention kernels, so it is the larger of theirs,
|err| <= 2^-8 |out| + (2^-11 + 2^-13 + 2^-16) A (1 + 2^-8), A = sum p |v| (weights rounded once to f16: 2^-11; what Q's
two e4m3 terms lose: 2^-13 for scores of order 1; sums and exp2: 2^-16; the output once to bf16: 2^-8), plus what weights
below f16's normal range add (``smallest_weights``)."""
from types import SimpleNamespace

import pytest
import torch

from tests.fp8_cache import E4M3, as_values, attention, orc, smallest_weights

pytestmark = pytest.mark.gpu

N_Q, N_KV, HD = 8, 2, 128
SCALE = HD ** -0.5


def _model(n_kv=N_KV, layers=2, w=None):
    cfg = SimpleNamespace(head_dim=HD, num_layers=layers, rms_eps=1e-6)
    return SimpleNamespace(cfg=cfg, n_q_local=N_Q, n_kv_local=n_kv, w=w or {},
                           layer_prefix=lambda i: f"model.layers.{i}.", device=torch.device("cuda"),
                           dtype=torch.bfloat16, ATTENTION_FAMILY="gqa", _gqa_b200_kv_dtype=E4M3)


def _build(mode, blocks, bs, **kw):
    from auto_infer_b200 import registry
    return registry.build_attention_backend(_model(**kw), mode, blocks, bs)


def _rows(g, t, heads):
    return torch.randn(t, heads, HD, generator=g).to(torch.bfloat16)


def _expect_cache(cache, before, k, v, slots):
    """``cache`` (on the GPU) holds what the write of k / v into ``before`` is defined to leave."""
    for codes, scale, old_codes, old_scale, rows in ((cache[0], cache[2], before[0], before[2], k),
                                                     (cache[1], cache[3], before[1], before[3], v)):
        want, want_scale = as_values(old_codes), old_scale.double()
        orc.write_kv_fp8(rows, want, want_scale, slots)
        assert torch.equal(scale.cpu().double(), want_scale)
        assert torch.equal(as_values(codes), want)


def _expect_output(got, q, cache, table, cu, kv):
    kc, vc, ks, vs = (x.cpu() for x in cache)
    want, _ = attention(q, kc, vc, ks, vs, table, cu, kv, SCALE)
    a, _ = attention(q, kc, vc.float().abs().to(vc.dtype), ks, vs, table, cu, kv, SCALE)
    tol = 2.0 ** -8 * want.abs() + (1 + 2.0 ** -8) * ((2.0 ** -11 + 2.0 ** -13 + 2.0 ** -16) * a + smallest_weights(
        q, kc, vc, ks, vs, table, cu, kv, SCALE))
    n = cu[-1]
    err = (got.cpu().double() - want)[:n].abs()
    assert (err <= tol[:n]).all(), float((err / tol[:n].clamp_min(1e-300)).max())


class _Requests:
    """Growing sequences over a shuffled pool; a finished one's pages are handed out again."""

    def __init__(self, g, blocks, bs):
        self.free, self.bs, self.pages, self.len = torch.randperm(blocks, generator=g).tolist(), bs, {}, {}

    def step(self, news):
        """news: {request: new tokens}; returns (slots, table, cu, kv)."""
        slots, cu, kv = [], [], []
        for r, n in news.items():
            have, pages = self.len.get(r, 0), self.pages.setdefault(r, [])
            while len(pages) * self.bs < have + n:
                pages.append(self.free.pop())
            slots += [pages[p // self.bs] * self.bs + p % self.bs for p in range(have, have + n)]
            self.len[r] = have + n
            cu.append(n + (cu[-1] if cu else 0))
            kv.append(have + n)
        table = torch.zeros(len(news), max(len(self.pages[r]) for r in news), dtype=torch.int32)
        for i, r in enumerate(news):
            table[i, :len(self.pages[r])] = torch.tensor(self.pages[r], dtype=torch.int32)
        return slots, table, cu, kv

    def finish(self, r):
        self.free += self.pages.pop(r)
        del self.len[r]


@pytest.mark.parametrize("bs", [16, 128])
def test_a_run_of_steps(bs):
    """Prompts, decode steps, verify rows, mixed steps, a request that ends and whose pages serve the next."""
    from auto_infer_b200 import ops
    from auto_infer_b200.forward_context import ForwardContext
    g = torch.Generator().manual_seed(bs)
    blocks = 12 if bs == 128 else 64
    backend, caches = _build("paged", blocks, bs)
    req = _Requests(g, blocks, bs)
    steps = [{"a": 1}, {"a": 37, "b": 150}, {"a": 1, "b": 1}, {"a": 1, "b": 1, "c": 90}, {"a": 4, "b": 2, "c": 1},
             "a", {"d": 200, "b": 1}, {"b": 1, "c": 33, "d": 1}, {"b": 5, "d": 1}, {"c": 1}]
    for news in steps:
        if isinstance(news, str):
            req.finish(news)
            continue
        slots, table, cu, kv = req.step(news)
        ctx = ForwardContext(None, None, torch.tensor(slots, dtype=torch.int32).cuda(), table.cuda(), cu, kv, None,
                             backend, caches, False)
        for layer in range(2):
            q, k, v = _rows(g, cu[-1], N_Q), _rows(g, cu[-1], N_KV) * (layer + 1), _rows(g, cu[-1], N_KV)
            before = [x.cpu() for x in caches[layer]]
            out = backend.paged_attention(layer, q.cuda(), k.cuda(), v.cuda(), ctx)
            torch.cuda.synchronize()
            assert ops.read_status("cuda") == 0
            _expect_cache(caches[layer], before, k, v, slots)
            _expect_output(out, q, caches[layer], table, cu, kv)


def test_both_kernels_side_by_side(monkeypatch):
    """A mixed step on disjoint SMs, over several rounds on one pooled plan."""
    from auto_infer_b200 import metadata, ops
    from auto_infer_b200.forward_context import ForwardContext
    monkeypatch.setattr(metadata, "mixed_split", lambda *a: 40)
    g = torch.Generator().manual_seed(1)
    backend, caches = _build("paged", 40, 64, layers=1)
    req = _Requests(g, 40, 64)
    for news in ({"a": 300}, {"a": 1, "b": 260}, {"a": 1, "b": 1, "c": 129}):
        slots, table, cu, kv = req.step(news)
        ctx = ForwardContext(None, None, torch.tensor(slots, dtype=torch.int32).cuda(), table.cuda(), cu, kv, None,
                             backend, caches, False)
        q, k, v = _rows(g, cu[-1], N_Q), _rows(g, cu[-1], N_KV), _rows(g, cu[-1], N_KV)
        out = backend.paged_attention(0, q.cuda(), k.cuda(), v.cuda(), ctx)
        torch.cuda.synchronize()
        assert ops.read_status("cuda") == 0
        assert backend._meta_pool and all(m.prefill_ctas == 40 for m in backend._meta_pool.values())
        _expect_output(out, q, caches[0], table, cu, kv)


@pytest.mark.parametrize("norm", [False, True])
def test_whole_sub_block(norm):
    """``attention()`` is the projection, the prologue (whose q and k are those of the 16-bit path, bit for bit), the
    slot write, the attention kernels and o_proj."""
    from auto_infer_b200 import ops
    from auto_infer_b200.forward_context import ForwardContext
    g = torch.Generator().manual_seed(7 + norm)
    hidden, t = 256, 45
    p = "model.layers.0.self_attn."
    w = {p + "qkv_proj.weight": torch.randn((N_Q + 2 * N_KV) * HD, hidden, generator=g) * 0.08,
         p + "qkv_proj.bias": torch.randn((N_Q + 2 * N_KV) * HD, generator=g) * 0.05,
         p + "o_proj.weight": torch.randn(hidden, N_Q * HD, generator=g) * 0.05}
    if norm:
        w |= {p + "q_norm.weight": torch.rand(HD, generator=g) + 0.5, p + "k_norm.weight": torch.rand(HD, generator=g) + 0.5}
    w = {n: x.to(torch.bfloat16).cuda() for n, x in w.items()}
    backend, caches = _build("paged", 16, 16, layers=1, w=w)
    slots = torch.randperm(16, generator=g)[:3].repeat_interleave(16)[:t] * 16 + torch.arange(t) % 16
    table = (slots[::16] // 16).int()[None].cuda()
    x = torch.randn(t, hidden, generator=g).to(torch.bfloat16).cuda()
    ang = torch.arange(t)[:, None] / 10000.0 ** (torch.arange(0, HD, 2) / HD)
    cos, sin = (torch.cat([f(ang)] * 2, -1)[:, None].to(torch.bfloat16).cuda() for f in (torch.cos, torch.sin))
    ctx = ForwardContext(None, None, slots.int().cuda(), table, [t], [t], None, backend, caches, False, cos=cos, sin=sin)
    got = backend.attention(0, x, ctx)

    q, k, v = (x @ w[p + "qkv_proj.weight"].t() + w[p + "qkv_proj.bias"]).split((N_Q * HD, N_KV * HD, N_KV * HD), -1)
    q, k, v = q.view(t, N_Q, HD), k.view(t, N_KV, HD), v.view(t, N_KV, HD)
    wide = torch.zeros(2, 16, 16, N_KV, HD, dtype=torch.bfloat16, device="cuda")
    kw = dict(q_norm_weight=w.get(p + "q_norm.weight"), k_norm_weight=w.get(p + "k_norm.weight"), eps=1e-6, want_k=True)
    q1, k1 = ops.gqa_rope_cache(q, k, v, cos, sin, wide[0], wide[1], slots.int().cuda(), **kw)
    q2, k2 = ops.gqa_rope_cache(q, k, v, cos, sin, None, None, None, **kw)
    assert torch.equal(q1, q2) and torch.equal(k1, k2)
    other, other_caches = _build("paged", 16, 16, layers=1)
    ctx2 = ForwardContext(None, None, slots.int().cuda(), table, [t], [t], None, other, other_caches, False)
    out = other.paged_attention(0, q1, k1, v, ctx2).reshape(t, -1) @ w[p + "o_proj.weight"].t()
    torch.cuda.synchronize()
    assert ops.read_status("cuda") == 0
    for a, b in zip(caches[0], other_caches[0]):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    assert torch.equal(got, out)
    _expect_cache(caches[0], [x.cpu() for x in _build("paged", 16, 16, layers=1)[1][0]], k1.cpu(), v.cpu(), slots.tolist())


def test_captured_gears_replay_for_other_lengths():
    """A decode gear and a prefill gear captured against the same caches, replayed in turn with eager steps in between."""
    from auto_infer_b200 import ops
    from auto_infer_b200.forward_context import ForwardContext
    g = torch.Generator().manual_seed(3)
    bs, blocks, rows, width = 16, 64, 4, 24
    backend, caches = _build("graph", blocks + rows, bs)

    class Gear:
        def __init__(self, tokens, seqs, cu, kv, slots):
            self.q, self.k, self.v = (torch.zeros(tokens, h, HD, dtype=torch.bfloat16, device="cuda") for h in (N_Q, N_KV, N_KV))
            self.slots = torch.tensor(slots, dtype=torch.int32).cuda()
            self.table = torch.arange(blocks, blocks + seqs, dtype=torch.int32).remainder(blocks + rows)[:, None].repeat(1, width).cuda()
            ctx = self.ctx(cu, kv)
            self.run(ctx)                               # the plan's buffers come to life
            torch.cuda.synchronize()
            self.graph = torch.cuda.CUDAGraph()
            backend.begin_capture()
            with torch.cuda.graph(self.graph):
                self.out = self.run(ctx)
            backend.end_capture()
            self.reg = backend.reg

        def ctx(self, cu, kv):
            return ForwardContext(None, None, self.slots, self.table, cu, kv, None, backend, caches, False)

        def run(self, ctx):
            return [backend.paged_attention(i, self.q, self.k, self.v, ctx) for i in range(2)]

    decode = Gear(rows, rows, list(range(1, rows + 1)), [1] * rows, [(blocks + i) * bs for i in range(rows)])
    wide = Gear(48, 6, [48] * 6, [48] + [0] * 5, [(blocks + i // bs) * bs + i % bs for i in range(48)])
    perm = torch.randperm(blocks, generator=g).tolist()
    turns = [(decode, [(1, 6), (1, 18)]), (wide, [(30, 130), (18, 18)]), (decode, [(1, 1), (1, 301), (1, 64), (1, 17)]),
             (wide, [(1, 90), (1, 17), (2, 40), (44, 108)]), (wide, [(8, 8 + 20 * i) for i in range(6)]), (decode, [(1, bs * width)])]
    for gear, seqs in turns:
        tokens, n = gear.q.shape[0], gear.table.shape[0]
        table, slots, cu, kv, at = torch.zeros(n, width, dtype=torch.int32), [], [], [], 0
        for b in range(n):
            if b < len(seqs):
                new, length = seqs[b]
                pages = perm[at:at + -(-length // bs)]
                at += len(pages)
            elif gear is decode:                        # a padding row on its own scratch block
                new, length, pages = 1, 1, [blocks + b]
            else:
                new, length, pages = 0, 0, []
            table[b, :len(pages)] = torch.tensor(pages, dtype=torch.int32)
            slots += [pages[p // bs] * bs + p % bs for p in range(length - new, length)]
            cu.append(new + (cu[-1] if cu else 0))
            kv.append(length)
        q, k, v = _rows(g, tokens, N_Q), _rows(g, tokens, N_KV), _rows(g, tokens, N_KV)
        for dst, src in ((gear.q, q), (gear.k, k), (gear.v, v), (gear.slots, torch.tensor(slots)), (gear.table, table)):
            dst.copy_(src)
        # pages a sequence has from before this step: fill them through the operator, eagerly
        old = [perm[i] * bs + j for i in range(at) for j in range(bs)]
        for i in range(2):
            ops.reshape_and_cache_fp8(_rows(g, len(old), N_KV).cuda(), _rows(g, len(old), N_KV).cuda(), *caches[i],
                                      torch.tensor(old, dtype=torch.int32).cuda())
        before = [[x.cpu() for x in cache] for cache in caches]
        backend.update_registrations(gear.reg, gear.ctx(cu, kv))
        gear.graph.replay()
        torch.cuda.synchronize()
        assert ops.read_status("cuda") == 0
        for i in range(2):
            _expect_cache(caches[i], before[i], k, v, slots)
            _expect_output(gear.out[i], q, caches[i], table, cu, kv)


@pytest.mark.parametrize("n_kv", [1, 3, 4])
def test_pages_move_with_their_scales(n_kv):
    """A prefill instance's blocks copied to a decode instance, to other block ids: codes and scales arrive unchanged (the
    scales of a page are 4 n_kv bytes, not always a multiple of 16), other pages stay."""
    from auto_infer_b200 import ops
    g = torch.Generator().manual_seed(n_kv)

    def pool(blocks):
        codes = lambda: torch.randint(0, 256, (blocks, 32, n_kv, HD), generator=g, dtype=torch.uint8).cuda().view(E4M3)
        return codes(), codes(), torch.rand(blocks, n_kv, generator=g).cuda(), torch.rand(blocks, n_kv, generator=g).cuda()

    src, dst = pool(9), pool(15)
    want = [x.cpu() for x in dst]
    ops.copy_blocks([src], [dst], [8, 0, 3], target_block_ids=[2, 14, 5])
    torch.cuda.synchronize()
    for a, b in zip(src, want):
        b.view(torch.uint8)[[2, 14, 5]] = a.cpu().view(torch.uint8)[[8, 0, 3]]
    for a, b in zip(dst, want):
        assert torch.equal(a.cpu().view(torch.uint8), b.view(torch.uint8))
    with pytest.raises(ValueError, match="types must match"):
        ops.copy_blocks([src], [tuple(x.to(torch.bfloat16) for x in src)], [1])
    assert ops.read_status("cuda") == 0
