"""Test helper: 8-bit paged caches with shuffled pages, and their values in 64 bits."""
import math

import torch

from oracle import paged_attention_oracle as orc

E4M3 = torch.float8_e4m3fn


def as_values(codes):
    """The numbers e4m3 codes stand for, float64 on the CPU."""
    return codes.cpu().float().double()


def empty_pool(blocks, bs, n_kv, fill_byte=0, scale=0.0, d=128):
    codes = torch.full((blocks, bs, n_kv, d), fill_byte, dtype=torch.uint8).view(E4M3)
    return codes, torch.full((blocks, n_kv), scale, dtype=torch.float32)


def random_pool(g, blocks, bs, n_kv, d=128, spread=1.0, any_scale=False):
    """Codes of random rows under page scales that vary by 2^(+-spread) or so; ``any_scale``: the
    scales are not powers of two."""
    x = torch.randn(blocks, bs, n_kv, d, generator=g, dtype=torch.float64) * 60
    scale = torch.exp2(torch.round(torch.randn(blocks, n_kv, generator=g) * spread) - 6)
    if any_scale:
        scale *= 1 + torch.rand(blocks, n_kv, generator=g)
    return x.clamp(-448, 448).to(torch.float32).to(E4M3), scale.float()


def deal_pages(g, lens, bs, spare=3):
    """(number of blocks, (B, max pages) block table, flat slots of all positions in order)."""
    need = [-(-n // bs) for n in lens]
    blocks = sum(need) + spare
    order = torch.randperm(blocks, generator=g)
    table = torch.zeros(len(lens), max(need + [1]), dtype=torch.int32)
    at, slots = 0, []
    for b, n in enumerate(need):
        pages = order[at:at + n]
        table[b, :n] = pages.int()
        at += n
        pos = torch.arange(lens[b])
        slots.append(pages[pos // bs] * bs + pos % bs)
    return blocks, table, slots


def attention(q, kc, vc, ks, vs, table, cu, kv_lens, scale, causal_base=None):
    """softmax(scale q (k s_k)) (v s_v) per row in 64 bits: (out, lse); a row that sees no key is 0 / -inf."""
    t, n_q, d = q.shape
    bs, n_kv = kc.shape[1], kc.shape[2]
    group = n_q // n_kv
    out = torch.zeros(t, n_q, d, dtype=torch.float64)
    lse = torch.full((t, n_q), -float("inf"), dtype=torch.float64)
    q0 = 0
    for b, end in enumerate(cu):
        n, k_len = end - q0, kv_lens[b]
        pages = table[b, :-(-k_len // bs)].long()
        base = k_len - n if causal_base is None else causal_base[b]
        for h in range(n_kv):
            k = (as_values(kc[pages, :, h]) * ks[pages, h].double()[:, None, None]).reshape(-1, d)[:k_len]
            v = (as_values(vc[pages, :, h]) * vs[pages, h].double()[:, None, None]).reshape(-1, d)[:k_len]
            for i in range(n):
                seen = max(0, min(base + i + 1, k_len))
                if not seen:
                    continue
                heads = slice(h * group, (h + 1) * group)
                s = q[q0 + i, heads].double() @ k[:seen].T * scale
                lse[q0 + i, heads] = torch.logsumexp(s, -1)
                out[q0 + i, heads] = torch.softmax(s, -1) @ v[:seen]
        q0 = end
    return out, lse


def smallest_weights(q, kc, vc, ks, vs, table, cu, kv_lens, scale, causal_base=None):
    """2^-25 W sum_j |cv_j| per output element, W = max_j p_j s_v,j over the keys j a row sees.

    What rounding the weights to f16 costs below f16's normal range.  A weight is taken relative to a
    reference R <= W (the running maximum of p_j s_v,j, or one up to 2^8 below it), w_j = p_j s_v,j / R.  f16 is off
    by at most half a step: 2^-11 w_j (half of 2^-10, and less) for w_j >= 2^-14, 2^-25 below.  The latter adds
    at most 2^-25 R |cv_j| per key to a row's output, which is at most 2^-25 W sum_j |cv_j|.  It only shows where
    the keys that carry the row have codes near 0 in a column."""
    t, n_q, d = q.shape
    bs, n_kv = kc.shape[1], kc.shape[2]
    group = n_q // n_kv
    out = torch.zeros(t, n_q, d, dtype=torch.float64)
    q0 = 0
    for b, end in enumerate(cu):
        n, k_len = end - q0, kv_lens[b]
        pages = table[b, :-(-k_len // bs)].long()
        base = k_len - n if causal_base is None else causal_base[b]
        for h in range(n_kv):
            k = (as_values(kc[pages, :, h]) * ks[pages, h].double()[:, None, None]).reshape(-1, d)[:k_len]
            codes = as_values(vc[pages, :, h]).reshape(-1, d)[:k_len].abs()
            s_v = vs[pages, h].double().repeat_interleave(bs)[:k_len]
            for i in range(n):
                seen = max(0, min(base + i + 1, k_len))
                if not seen:
                    continue
                heads = slice(h * group, (h + 1) * group)
                p = torch.softmax(q[q0 + i, heads].double() @ k[:seen].T * scale, -1)
                top = (p * s_v[:seen]).amax(-1, keepdim=True)
                out[q0 + i, heads] = 2.0 ** -25 * top * codes[:seen].sum(0)
        q0 = end
    return out


def sink_case(seed, lens, q_lens, n_q, bs, mass, sink_v):
    """Rows whose first key takes the share ``mass`` of the softmax over a long context and has a V of ``sink_v`` times
    the others' size (0: of zeros), so that the row's output is made of many weights, each far below that key's.  One kv
    head; half of V's columns are of one sign.  Same tuple as the kernel tests' cases."""
    g = torch.Generator().manual_seed(seed)
    blocks, table, _ = deal_pages(g, lens, bs)
    kc, ks = random_pool(g, blocks, bs, 1, spread=0.0)
    vc, vs = random_pool(g, blocks, bs, 1, spread=0.0)
    kx, vx = kc.float(), vc.float()
    kx[..., 0] = 0.0
    vx[..., ::2] = vx[..., ::2].abs()
    for b in range(len(lens)):
        page = int(table[b, 0])
        kx[page, 0] = 0.0
        kx[page, 0, 0, 0] = 448.0
        vx[page, 0] *= sink_v
    cu = torch.tensor(q_lens).cumsum(0).tolist()
    q = torch.randn(cu[-1], n_q, 128, generator=g)
    scale, at = 128 ** -0.5, 0
    for n, end in zip(lens, cu):
        # the other scores are about N(0, 1): their sum is about n exp(1/2)
        gap = math.log(mass / (1 - mass)) + math.log(max(n - 1, 1)) + 0.5
        q[at:end, :, 0] = gap / (scale * 448.0 * float(ks[0, 0]))
        at = end
    return q.to(torch.bfloat16), kx.to(E4M3), vx.to(E4M3), ks, vs, table, cu, list(lens), scale


__all__ = ["sink_case", "smallest_weights", "E4M3", "as_values", "empty_pool", "random_pool", "deal_pages", "attention", "orc"]
