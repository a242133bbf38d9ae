"""Workloads of the 8-bit paged KV cache: what is measured of its three operators.

The cache holds K and V as e4m3 codes in pages of ``block_size`` tokens, with one fp32 scale per
(page, kv head), K and V apart; a value is its code times its page's scale.

* ``write``    ``ops.reshape_and_cache_fp8``: a step's new K / V rows are quantised into their slots.
  Per page, head and call: the scale is the smallest power of two that brings the largest magnitude
  of the new rows within 448; a page whose first slot is written starts anew with it, any other page
  keeps the larger of it and its own, and when the scale grows its other rows are rounded to it again.
* ``decode``   ``ops.paged_decode_gqa_fp8``: attention of decode / verify rows (q_len * group <= 16).
* ``prefill``  ``ops.paged_prefill_gqa_fp8``: attention of wide query blocks over a cached prefix.

``own`` false: the plain form, elementary torch operations in fp32.  ``own`` true: the calls of the
framework.
"""
import math
import random

import torch

own = False

HEAD_DIM = 128
E4M3 = torch.float8_e4m3fn
E4M3_MAX = 448.0


# ----------------------------------------------------------------------------- cases
def listed():
    return [
        # one decode step's rows, a batch of 16 (16 q / 8 kv heads): the smallest write, latency counts
        dict(name="write decode step", op="write", n_kv=8, block_size=128, lens_seed=1, seqs=16, q_lo=1, q_hi=1,
             kv_lo=512, kv_hi=2048, chunks=0, chunk=0, prefix_hi=0),
        # a mixed step: 60 decode rows and four 512-token chunks over cached prefixes
        dict(name="write mixed step", op="write", n_kv=8, block_size=128, lens_seed=2, seqs=60, q_lo=1, q_hi=1,
             kv_lo=256, kv_hi=8192, chunks=4, chunk=512, prefix_hi=4096),
        # one long prompt chunk with small pages and an odd length
        dict(name="write long chunk", op="write", n_kv=8, block_size=16, lens_seed=3, seqs=0, q_lo=1, q_hi=1,
             kv_lo=1, kv_hi=1, chunks=1, chunk=8191, prefix_hi=100),
        # one sequence, short context: a single user's token, pure latency
        dict(name="decode single", op="decode", n_q=16, n_kv=8, block_size=128, lens_seed=4, seqs=1, q_lo=1, q_hi=1,
             kv_lo=777, kv_hi=777, lse=False),
        # batch 16, contexts of a chat (16 q / 8 kv heads)
        dict(name="decode batch 16", op="decode", n_q=16, n_kv=8, block_size=128, lens_seed=5, seqs=16, q_lo=1, q_hi=1,
             kv_lo=512, kv_hi=2048, lse=False),
        # verification of one drafted token: two query rows a sequence, with the log-sum-exp that merges want
        dict(name="decode verify", op="decode", n_q=32, n_kv=8, block_size=128, lens_seed=6, seqs=16, q_lo=2, q_hi=2,
             kv_lo=512, kv_hi=4096, lse=True),
        # 60 ragged sequences on small pages
        dict(name="decode ragged 60", op="decode", n_q=32, n_kv=8, block_size=16, lens_seed=7, seqs=60, q_lo=1, q_hi=1,
             kv_lo=256, kv_hi=8192, lse=False),
        # long-context decode: 8 sequences of 131072 tokens (64 q / 8 kv heads)
        dict(name="decode 8 x 131072", op="decode", n_q=64, n_kv=8, block_size=128, lens_seed=8, seqs=8, q_lo=1, q_hi=1,
             kv_lo=131072, kv_hi=131072, lse=False),
        # short drafts too wide for the decode form: a handful of rows over cached contexts
        dict(name="prefill draft 5", op="prefill", n_q=32, n_kv=8, block_size=128, lens_seed=9, seqs=16, q_lo=5, q_hi=5,
             kv_lo=512, kv_hi=4096),
        # four 512-token chunks over cached prefixes
        dict(name="prefill chunks", op="prefill", n_q=32, n_kv=8, block_size=128, lens_seed=10, seqs=4, q_lo=512, q_hi=512,
             kv_lo=512, kv_hi=4608),
        # odd chunk lengths, small pages, a group that does not divide the 128-row tile
        dict(name="prefill odd", op="prefill", n_q=28, n_kv=4, block_size=32, lens_seed=11, seqs=3, q_lo=301, q_hi=777,
             kv_lo=1001, kv_hi=2999),
        # one prompt of 8192 tokens
        dict(name="prefill prompt 8192", op="prefill", n_q=32, n_kv=8, block_size=128, lens_seed=12, seqs=1, q_lo=8192,
             q_hi=8192, kv_lo=8192, kv_hi=8192),
    ]


def _between(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["write", "decode", "decode", "prefill"])
    n_kv = rng.choice([1, 2, 4, 8])
    block_size = rng.choice([16, 32, 64, 128, 256])
    seed = rng.randrange(1 << 20)
    if op == "write":
        chunks = rng.choice([0, 0, 1, 2, 3])
        return dict(op=op, n_kv=n_kv, block_size=block_size, lens_seed=seed,
                    seqs=_between(rng, 1, 128), q_lo=1, q_hi=rng.choice([1, 1, 2, 4]), kv_lo=4, kv_hi=_between(rng, 16, 4096),
                    chunks=chunks, chunk=_between(rng, 17, 2600) if chunks else 0,
                    prefix_hi=_between(rng, 1, 2000) if chunks else 0)
    if op == "decode":
        group = rng.choice([1, 2, 3, 4, 5, 7, 8, 16])
        seqs = _between(rng, 1, 64)
        hi = _between(rng, 2, min(131072, 1000000 // seqs))
        lo = _between(rng, 1, hi)
        return dict(op=op, n_q=n_kv * group, n_kv=n_kv, block_size=block_size, lens_seed=seed, seqs=seqs, q_lo=1,
                    q_hi=rng.randint(1, max(1, min(4, 16 // group, lo))), kv_lo=lo, kv_hi=hi, lse=rng.random() < 0.3)
    group = rng.choice([1, 2, 3, 4, 5, 7, 8, 16])
    seqs = _between(rng, 1, 8)
    q_hi = _between(rng, 17, max(18, 4096 // seqs))
    q_lo = _between(rng, 17, q_hi)
    kv_lo = q_hi + _between(rng, 1, 200) - 1
    return dict(op=op, n_q=n_kv * group, n_kv=n_kv, block_size=block_size, lens_seed=seed, seqs=seqs, q_lo=q_lo, q_hi=q_hi,
                kv_lo=kv_lo, kv_hi=kv_lo + _between(rng, 1, 3000))


def _lengths(case):
    """(query lengths, total kv lengths, step's tokens included) of the case's sequences."""
    r = random.Random(case["lens_seed"])
    q, kv = [], []
    for _ in range(case["seqs"]):
        n = r.randint(case["q_lo"], case["q_hi"])
        q.append(n)
        kv.append(max(n, r.randint(case["kv_lo"], case["kv_hi"])))
    for _ in range(case.get("chunks", 0)):
        q.append(case["chunk"])
        kv.append(case["chunk"] + r.randint(0, case["prefix_hi"]))
    return q, kv


def work(case):
    q, kv = _lengths(case)
    t, n_kv, bs = sum(q), case["n_kv"], case["block_size"]
    if case["op"] == "write":
        pages = sum((k - 1) // bs - (k - n) // bs + 1 for n, k in zip(q, kv))
        # rows read in 16 bits and written in 8, K and V; slots; the touched pages' scales read and written
        return dict(bytes=2 * t * n_kv * HEAD_DIM * 3 + 4 * t + 2 * 2 * 4 * pages * n_kv, flops=2 * 2 * t * n_kv * HEAD_DIM)
    n_q = case["n_q"]
    pages = sum(-(-k // bs) for k in kv)
    seen = sum(n * k - n * (n - 1) // 2 for n, k in zip(q, kv))            # (query token, visible key) pairs
    return dict(bytes=2 * sum(kv) * n_kv * HEAD_DIM + 2 * 4 * pages * n_kv + 4 * pages + 2 * 2 * t * n_q * HEAD_DIM,
                flops=4 * HEAD_DIM * n_q * seen)


# ----------------------------------------------------------------------------- inputs
def _paged_codes(g, blocks, bs, n_kv):
    """A filled cache: codes and scales of rows whose size varies by channel and by page, as keys' do."""
    dev = "cuda"
    channel = torch.exp(0.5 * torch.randn(n_kv, HEAD_DIM, generator=g, device=dev))
    codes = torch.empty(blocks, bs, n_kv, HEAD_DIM, dtype=E4M3, device=dev)
    scales = torch.empty(blocks, n_kv, dtype=torch.float32, device=dev)
    step = max(1, (1 << 27) // (bs * n_kv * HEAD_DIM))
    for b in range(0, blocks, step):
        n = min(step, blocks - b)
        x = torch.randn(n, bs, n_kv, HEAD_DIM, generator=g, device=dev) * channel
        x *= torch.exp(0.3 * torch.randn(n, 1, n_kv, 1, generator=g, device=dev))
        mant, exp = torch.frexp(x.abs().amax(dim=(1, 3)))
        s = torch.ldexp(torch.ones_like(mant), exp - 9 + (mant > 0.875).int())
        codes[b:b + n] = (x / s[:, None, :, None]).to(E4M3)
        scales[b:b + n] = s
    return codes, scales


def prepare(case, seed):
    dev = "cuda"
    g = torch.Generator(device=dev).manual_seed(seed)
    q, kv = _lengths(case)
    bs, n_kv = case["block_size"], case["n_kv"]
    need = [-(-k // bs) for k in kv]
    blocks = sum(need) + 3
    order = torch.randperm(blocks, generator=g, device=dev).to(torch.int32)
    table = torch.zeros(len(kv), max(need), dtype=torch.int32, device=dev)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    kc, ks = _paged_codes(g, blocks, bs, n_kv)
    vc, vs = _paged_codes(g, blocks, bs, n_kv)
    cu = []
    for n in q:
        cu.append((cu[-1] if cu else 0) + n)
    s = dict(case=case, key_cache=kc, value_cache=vc, key_scale=ks, value_scale=vs, block_table=table)
    t = cu[-1]
    if case["op"] == "write":
        where = torch.cat([torch.arange(k - n, k, device=dev) for n, k in zip(q, kv)])
        seq = torch.repeat_interleave(torch.arange(len(q), device=dev), torch.tensor(q, device=dev))
        s["slots"] = (table[seq, where // bs] * bs + (where % bs).to(torch.int32)).to(torch.int32)
        # rows as views of a packed projection; now and then a token larger than its page's rows so far
        kv_rows = torch.randn(t, 2 * n_kv * HEAD_DIM, generator=g, device=dev)
        kv_rows *= torch.exp(0.5 * torch.randn(t, 1, generator=g, device=dev))
        kv_rows = kv_rows.to(torch.bfloat16)
        s["key"] = kv_rows[:, :n_kv * HEAD_DIM].view(t, n_kv, HEAD_DIM)
        s["value"] = kv_rows[:, n_kv * HEAD_DIM:].view(t, n_kv, HEAD_DIM)
        return s
    n_q = case["n_q"]
    s["scale"] = HEAD_DIM ** -0.5
    s["q"] = torch.randn(t, n_q, HEAD_DIM, generator=g, device=dev).to(torch.bfloat16)
    s["lse"] = torch.empty(t, n_q, dtype=torch.float32, device=dev) if case.get("lse") else None
    # the step's lengths as a user's program has them: on the host for the plan, on the device for the plain form
    s["q_len"], s["kv_len"] = torch.tensor(q, device=dev), torch.tensor(kv, device=dev)
    s["q_max"] = max(q)
    if own:
        from auto_infer_b200 import ops
        s["plan"] = (ops.DecodePlan(cu, kv, n_q, n_kv, dev) if case["op"] == "decode"
                     else ops.PrefillPlan(cu, kv, n_q, n_kv, dev))
    return s


# ----------------------------------------------------------------------------- the passes
def run(state):
    op = state["case"]["op"]
    if own:
        from auto_infer_b200 import ops
        caches = (state["key_cache"], state["value_cache"], state["key_scale"], state["value_scale"])
        if op == "write":
            ops.reshape_and_cache_fp8(state["key"], state["value"], *caches, state["slots"])
            return dict(zip(("key_cache", "value_cache", "key_scale", "value_scale"), caches))
        if op == "decode":
            out = ops.paged_decode_gqa_fp8(state["q"], *caches, state["block_table"], state["plan"], state["scale"],
                                           lse_out=state["lse"])
        else:
            out = ops.paged_prefill_gqa_fp8(state["q"], *caches, state["block_table"], state["plan"], state["scale"])
        return dict(out=out) if state.get("lse") is None else dict(out=out, lse=state["lse"])
    if op == "write":
        _plain_write(state["key"], state["key_cache"], state["key_scale"], state["slots"])
        _plain_write(state["value"], state["value_cache"], state["value_scale"], state["slots"])
        return {n: state[n] for n in ("key_cache", "value_cache", "key_scale", "value_scale")}
    out, lse = _plain_attention(state)
    return dict(out=out, lse=lse) if state.get("lse") is not None else dict(out=out)


def _plain_write(rows, cache, scale, slots):
    bs = cache.shape[1]
    slots = slots.long()
    off = slots % bs
    pages, of = torch.unique(slots // bs, return_inverse=True)
    x = rows.float()
    top = torch.zeros(len(pages), x.shape[1], device=x.device).index_reduce_(0, of, x.abs().amax(-1), "amax")
    mant, exp = torch.frexp(top)                     # top = mant * 2^exp, mant in [0.5, 1), and 448 = 0.875 * 2^9
    call = torch.ldexp(torch.ones_like(top), (exp - 9 + (mant > 0.875).int()).clamp_min(-126))
    anew = torch.zeros(len(pages), device=x.device).index_reduce_(0, of, (off == 0).float(), "amax")[:, None] > 0
    old = scale[pages]
    s = torch.where(anew, call, torch.maximum(old, call))
    ratio = torch.where(anew, torch.ones_like(s), old / s)
    codes = cache.view(torch.uint8)
    page = codes[pages].view(E4M3).float() * ratio[:, None, :, None]
    codes[pages] = page.to(E4M3).view(torch.uint8)
    codes[pages[of], off] = (x / s[of][:, :, None]).to(E4M3).view(torch.uint8)
    scale[pages] = s


def _plain_rows(cache, scale, table):
    """The sequences' cached rows in fp32, (B, Hkv, tokens, D)."""
    t = table.long()
    x = cache.view(torch.uint8)[t].view(E4M3).float() * scale[t][:, :, None, :, None]
    return x.flatten(1, 2).transpose(1, 2)


def _plain_attention(state):
    q, table, q_len, kv_len = state["q"], state["block_table"], state["q_len"], state["kv_len"]
    n_kv = state["key_cache"].shape[2]
    n_q, dev = q.shape[1], q.device
    start = torch.cumsum(q_len, 0) - q_len
    i = torch.arange(state["q_max"], device=dev)
    have = i < q_len[:, None]                                                   # (B, L): a query token
    tok = torch.where(have, start[:, None] + i, 0)
    k = _plain_rows(state["key_cache"], state["key_scale"], table)
    qg = q.float()[tok].unflatten(2, (n_kv, n_q // n_kv)).permute(0, 2, 1, 3, 4).flatten(2, 3)   # (B, Hkv, L*G, D)
    scores = (qg @ k.transpose(2, 3)) * state["scale"]
    del k
    last = (kv_len - q_len)[:, None] + i                                        # last visible key of a query token
    hide = torch.arange(scores.shape[-1], device=dev) > torch.where(have, last, -1)[:, :, None]
    hide = hide[:, None, :, None, :].expand(-1, -1, -1, n_q // n_kv, -1).flatten(2, 3)
    scores.masked_fill_(hide, -math.inf)
    m = scores.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    p = torch.exp_(scores.sub_(m))
    l = p.sum(-1, keepdim=True)
    o = (p @ _plain_rows(state["value_cache"], state["value_scale"], table)) / torch.where(l > 0, l, 1.0)
    o = o.unflatten(2, (-1, n_q // n_kv)).permute(0, 2, 1, 3, 4).flatten(2, 3)  # (B, L, Hq, D)
    lse = (m + torch.log(l)).squeeze(-1).unflatten(2, (-1, n_q // n_kv)).permute(0, 2, 1, 3).flatten(2, 3)
    return o[have].to(q.dtype), lse[have]


# ----------------------------------------------------------------------------- from the definition, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "write":
        out = {}
        for name in ("key", "value"):
            out[name + "_cache"], out[name + "_scale"] = _exact_write(
                s[name].double(), s[name + "_cache"].double(), s[name + "_scale"].double(), s["slots"].tolist())
        return out
    q, kv = _lengths(case)
    n_kv, bs = case["n_kv"], case["block_size"]
    group = case["n_q"] // n_kv
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full(s["q"].shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    t0 = 0
    for b, (n, k) in enumerate(zip(q, kv)):
        pages = s["block_table"][b, :-(-k // bs)].long()
        for h in range(n_kv):
            keys, values = (
                (s[c + "_cache"].view(torch.uint8)[pages, :, h].view(E4M3).double()
                 * s[c + "_scale"][pages, h].double()[:, None, None]).reshape(-1, HEAD_DIM)[:k] for c in ("key", "value"))
            for lo in range(0, n, 2048):
                hi = min(n, lo + 2048)
                for head in range(h * group, (h + 1) * group):
                    x = s["q"][t0 + lo:t0 + hi, head].double() @ keys.T / math.sqrt(HEAD_DIM)
                    if n > 1:
                        seen = torch.arange(k, device="cuda")[None, :] <= torch.arange(k - n + lo, k - n + hi, device="cuda")[:, None]
                        x = x.masked_fill(~seen, -math.inf)
                    lse[t0 + lo:t0 + hi, head] = torch.logsumexp(x, -1)
                    out[t0 + lo:t0 + hi, head] = torch.exp(x - lse[t0 + lo:t0 + hi, head, None]) @ values
        t0 += n
    return dict(out=out, lse=lse) if case.get("lse") else dict(out=out)


def _exact_e4m3(x):
    """Nearest e4m3 value, ties to the even one: steps of 2^(e-3) for |x| in [2^e, 2^(e+1)), of 2^-9 below 2^-6."""
    e = torch.frexp(x.abs().clamp_min(2.0 ** -6)).exponent - 1
    step = torch.ldexp(torch.ones_like(x), e - 3)
    return torch.round(x / step) * step


def _exact_write(rows, cache, scale, slots):
    """Page by page; ``cache`` and ``scale`` in 64 bits, updated and returned."""
    bs = cache.shape[1]
    by_page = {}
    for t, slot in enumerate(slots):
        by_page.setdefault(slot // bs, {})[slot % bs] = t
    for page, taken in by_page.items():
        offs = torch.tensor(list(taken), device=rows.device)
        x = rows[torch.tensor(list(taken.values()), device=rows.device)]
        top = x.abs().amax(dim=(0, 2))
        call = torch.ldexp(torch.ones_like(top), torch.round(torch.log2(top / E4M3_MAX)).clamp(-125, 126).int())
        call = torch.where(E4M3_MAX * call < top, 2 * call, torch.where(E4M3_MAX * call / 2 >= top, call / 2, call))
        if 0 in taken:
            new = call
        else:
            new = torch.maximum(scale[page], call)
            grown = new > scale[page]
            again = _exact_e4m3(cache[page] * (scale[page] / new)[None, :, None])
            cache[page] = torch.where(grown[None, :, None], again, cache[page])
        cache[page, offs] = _exact_e4m3(x / new[None, :, None])
        scale[page] = new
    return cache, scale
