"""CPU oracle for the paged-attention path.  TEST INFRASTRUCTURE ONLY.

This module restates, in plain CPU torch, the arithmetic of auto-infer's
attention path so that the CUDA kernels can be checked against it.  It is a
checker: only the test-suite, the smoke entry point and the benchmark's CPU
baseline leg import it.  Nothing in the shipped package may call it.

Parity status: PINNED for the attention core, the GQA head mapping, the slot
mapping, the absorbed-MLA algebra, the non-absorbed MLA sub-block (K 192 / V 128 per head)
and the cache write against outputs of the
reference's own importable functions (committed fixtures, generated by
``tests/golden/make_golden.py``).  The vendor operators the reference calls on
its NPU (``torch_npu._npu_reshape_and_cache``,
``torch_npu.npu_fused_infer_attention_score``; torch_npu 2.10.0, unpinned in the
reference's pyproject.toml:9-11) are closed source and absent, so for those two
the pin is on the reference's call contract and on its eager path, not on the
vendor kernel's bits.

Reference anchors (paths inside the auto-infer project):
  * attention core ............ auto_infer/layers/attention/base.py:64-80
  * GQA head expansion ........ auto_infer/layers/attention/gqa.py:120-131
  * paged call contract ....... auto_infer/layers/attention/base.py:48-61
  * cache write contract ...... auto_infer/layers/attention/base.py:41-45
  * slot arithmetic ........... auto_infer/engine/token_layout.py:1-4
  * absorbed MLA .............. auto_infer/layers/attention/mla.py:67-73,105-121
  * non-absorbed MLA .......... auto_infer/layers/attention/mla.py:23-64,134-164
  * CP chunking convention .... auto_infer/models/qwen2.py:189-197
"""
from __future__ import annotations

import math

import torch


# --------------------------------------------------------------------------- #
# integer contracts (bit-exact)
# --------------------------------------------------------------------------- #
def slot_mapping(block_table, positions, block_size):
    """slot = block_table[pos // bs] * bs + pos % bs
    (auto_infer/engine/token_layout.py:1-4).  Works on ints, numpy arrays and
    torch tensors alike."""
    return block_table[positions // block_size] * block_size + positions % block_size


def write_kv(key, value, key_cache, value_cache, slots):
    """Scatter the step's K/V rows into the paged cache by flat slot index
    (call contract of auto_infer/layers/attention/base.py:41-45; callers
    gqa.py:76-79, mla.py:243-245).  key (T, Hkv, Dk), value (T, Hkv, Dv); caches
    (num_blocks, block_size, Hkv, D*).  Later rows win when slots repeat, as a
    sequential scatter does."""
    slots = torch.as_tensor(slots, dtype=torch.long)
    kc = key_cache.view(-1, key_cache.shape[-2], key_cache.shape[-1])
    kc[slots] = key
    if value is not None and value_cache is not None:
        vc = value_cache.view(-1, value_cache.shape[-2], value_cache.shape[-1])
        vc[slots] = value


def gather_paged(cache, block_row, kv_len):
    """Logical (kv_len, H, D) view of one sequence's cache rows through its
    block-table row.  Lengths, not zero entries, bound the walk: block 0 is a
    valid block (auto_infer/worker/model_runner.py:143,160)."""
    block_size = cache.shape[1]
    n_blocks = (kv_len + block_size - 1) // block_size
    ids = torch.as_tensor(block_row[:n_blocks], dtype=torch.long)
    pages = cache[ids]                                   # (n_blocks, bs, H, D)
    return pages.reshape(-1, cache.shape[2], cache.shape[3])[:kv_len]


# --------------------------------------------------------------------------- #
# attention core
# --------------------------------------------------------------------------- #
def _core_literal(q, k, v, scale):
    """The reference arithmetic for one sequence, q_len <= kv_len, bottom-right
    causal (key j visible to query row i iff j <= kv_len - q_len + i).

    q (q_len, H, D), k/v (kv_len, H, D*) already head-expanded.  Follows
    auto_infer/layers/attention/base.py:70-78 line by line: fp32 scores times
    scale plus an additive -inf mask, fp32 softmax, probabilities cast to the
    query dtype, then P @ V in that dtype.  Returns (out (q_len, H, Dv) in q's
    dtype, lse (q_len, H) fp32, natural log)."""
    q_len, kv_len = q.shape[0], k.shape[0]
    qh = q.transpose(0, 1)
    kh = k.transpose(0, 1)
    vh = v.transpose(0, 1)
    mask = torch.triu(
        torch.full((q_len, kv_len), float("-inf"), dtype=torch.float32),
        diagonal=kv_len - q_len + 1)
    scores = (qh.float() @ kh.float().transpose(-1, -2)) * scale + mask
    probability = torch.softmax(scores, dim=-1).to(q.dtype)
    out = (probability @ vh).transpose(0, 1)
    lse = torch.logsumexp(scores, dim=-1).transpose(0, 1)
    return out, lse


def _core_grouped(q, k, v, scale, kv_chunk=16384):
    """Same arithmetic without materialising the head-expanded K/V, for long
    contexts: query heads are folded into rows of their kv head and the keys are
    walked in chunks with a two-pass softmax (max first, then exp / sum), so the
    values equal the literal form up to fp32 summation order.  q (q_len, Hq, D),
    k/v (kv_len, Hkv, D*)."""
    q_len, n_q, d = q.shape
    kv_len, n_kv = k.shape[0], k.shape[1]
    group = n_q // n_kv
    dv = v.shape[-1]
    # rows ordered (kv head, q position, head-in-group)
    qg = q.view(q_len, n_kv, group, d).permute(1, 0, 2, 3).reshape(n_kv, q_len * group, d).float()
    limit = (kv_len - q_len + torch.arange(q_len)).repeat_interleave(group)  # last visible key

    def chunk_scores(start, stop):
        kc = k[start:stop].transpose(0, 1).float()                # (Hkv, c, D)
        s = (qg @ kc.transpose(-1, -2)) * scale                   # (Hkv, rows, c)
        idx = torch.arange(start, stop)
        s = s.masked_fill(idx[None, None, :] > limit[None, :, None], float("-inf"))
        return s

    row_max = torch.full((n_kv, q_len * group), float("-inf"))
    for start in range(0, kv_len, kv_chunk):
        row_max = torch.maximum(row_max, chunk_scores(start, min(kv_len, start + kv_chunk)).amax(-1))
    denom = torch.zeros_like(row_max)
    for start in range(0, kv_len, kv_chunk):
        denom += torch.exp(chunk_scores(start, min(kv_len, start + kv_chunk)) - row_max[..., None]).sum(-1)
    acc = torch.zeros(n_kv, q_len * group, dv)
    for start in range(0, kv_len, kv_chunk):
        stop = min(kv_len, start + kv_chunk)
        p = (torch.exp(chunk_scores(start, stop) - row_max[..., None]) / denom[..., None]).to(q.dtype)
        acc += (p @ v[start:stop].transpose(0, 1)).float()        # bf16 P @ V per chunk, fp32 across
    out = acc.view(n_kv, q_len, group, dv).permute(1, 0, 2, 3).reshape(q_len, n_q, dv).to(q.dtype)
    lse = (row_max + torch.log(denom)).view(n_kv, q_len, group).permute(1, 0, 2).reshape(q_len, n_q)
    return out, lse


def paged_attention(q, key_cache, value_cache, block_table, cu_seqlens_q, seqlens_kv,
                    scale, *, return_lse=False, literal_max_kv=4096, kv_ranges=None):
    """Paged attention with the reference's call contract
    (auto_infer/layers/attention/base.py:48-61): q (T, Hq, D) packed TND,
    caches (num_blocks, block_size, Hkv, D*), block_table (B, max_blocks),
    ``cu_seqlens_q`` cumulative, ``seqlens_kv`` per sequence and including the
    step's own tokens, bottom-right causal mask (sparse_mode 3).

    ``kv_ranges`` optionally restricts sequence b to keys [lo, hi) — the
    context-parallel slice of one rank; the mask still uses global positions.
    Sequences up to ``literal_max_kv`` keys use the literal reference form."""
    n_q = q.shape[1]
    n_kv = key_cache.shape[2]
    group = n_q // n_kv
    outs, lses = [], []
    start = 0
    for b, end in enumerate(cu_seqlens_q):
        kv_len = int(seqlens_kv[b])
        q_b = q[start:end]
        q_len = end - start
        if q_len == 0:
            continue
        k_b = gather_paged(key_cache, block_table[b], kv_len)
        v_b = gather_paged(value_cache, block_table[b], kv_len)
        if kv_ranges is not None:
            lo, hi = kv_ranges[b]
            out_b, lse_b = _core_range(q_b, k_b, v_b, scale, kv_len, lo, hi)
        elif kv_len <= literal_max_kv:
            out_b, lse_b = _core_literal(
                q_b, k_b.repeat_interleave(group, dim=1), v_b.repeat_interleave(group, dim=1), scale)
        else:
            out_b, lse_b = _core_grouped(q_b, k_b, v_b, scale)
        outs.append(out_b)
        lses.append(lse_b)
        start = end
    out = torch.cat(outs, dim=0)
    if return_lse:
        return out, torch.cat(lses, dim=0)
    return out


def _core_range(q, k, v, scale, kv_len, lo, hi):
    """Attention of one sequence restricted to keys [lo, hi) with the mask taken
    at global key positions — what one context-parallel rank computes.  Rows
    that see no key in the range return out = 0 and lse = -inf."""
    q_len, n_q, _ = q.shape
    group = n_q // k.shape[1]
    kk = k[lo:hi].repeat_interleave(group, dim=1).transpose(0, 1)
    vv = v[lo:hi].repeat_interleave(group, dim=1).transpose(0, 1)
    idx = torch.arange(lo, hi)
    limit = kv_len - q_len + torch.arange(q_len)
    mask = torch.zeros(q_len, hi - lo, dtype=torch.float32)
    mask.masked_fill_(idx[None, :] > limit[:, None], float("-inf"))
    scores = (q.transpose(0, 1).float() @ kk.float().transpose(-1, -2)) * scale + mask
    lse = torch.logsumexp(scores, dim=-1)
    empty = torch.isinf(lse) & (lse < 0)
    probability = torch.exp(scores - torch.where(empty, torch.zeros_like(lse), lse)[..., None])
    probability = torch.where(empty[..., None], torch.zeros_like(probability), probability).to(q.dtype)
    out = (probability @ vv).transpose(0, 1)
    return out, lse.transpose(0, 1)


# --------------------------------------------------------------------------- #
# log-sum-exp merge (split-KV and context-parallel partials)
# --------------------------------------------------------------------------- #
def lse_combine(o_parts, lse_parts, out_dtype=torch.bfloat16):
    """Merge normalised partial outputs: o = sum_r w_r o_r with
    w_r = exp(lse_r - lse), lse = logsumexp_r lse_r.  o_parts (R, rows, D) fp32,
    lse_parts (R, rows) fp32 (-inf marks an empty part).  Returns (o, lse)."""
    lse = torch.logsumexp(lse_parts, dim=0)
    safe = torch.where(torch.isinf(lse), torch.zeros_like(lse), lse)
    w = torch.exp(lse_parts - safe[None])
    w = torch.where(torch.isinf(lse_parts) & (lse_parts < 0), torch.zeros_like(w), w)
    o = (w[..., None] * o_parts.float()).sum(0)
    return o.to(out_dtype), lse


# --------------------------------------------------------------------------- #
# absorbed MLA (DeepSeek-V2/V3, Moonlight)
# --------------------------------------------------------------------------- #
def build_absorb_weights(kv_b_weight, num_heads, qk_nope, v_head_dim, kv_lora_rank):
    """kv_b_proj (H*(nope+vd), kvl) -> W_UK (H, nope, kvl), W_UV (H, vd, kvl)
    (auto_infer/layers/attention/mla.py:67-73)."""
    w = kv_b_weight.view(num_heads, qk_nope + v_head_dim, kv_lora_rank)
    w_uk, w_uv = w.split([qk_nope, v_head_dim], dim=1)
    return w_uk.contiguous(), w_uv.contiguous()


def mla_absorbed_attention(q_nope, q_pe, latent_cache, block_table, cu_seqlens_q,
                           seqlens_kv, scale, w_uk, w_uv, *, return_latent=False):
    """Absorbed-MLA attention after the projections
    (auto_infer/layers/attention/mla.py:105-121): the query is folded into the
    latent space with W_UK, one MQA head of width kvl+rope is attended with
    V = K, the first kvl output columns are kept and folded back with W_UV.
    latent_cache (num_blocks, block_size, 1, kvl+rope) holds [ckv | k_pe] per
    token (stored once; the reference stores it twice, mla.py:210-212, because
    its vendor op wants symmetric K and V)."""
    kvl = w_uk.shape[-1]
    q_absorbed = torch.einsum("tnp,npl->tnl", q_nope, w_uk)
    q_latent = torch.cat([q_absorbed, q_pe], dim=-1).contiguous()
    attn = paged_attention(q_latent, latent_cache, latent_cache, block_table,
                           cu_seqlens_q, seqlens_kv, scale)
    o_latent = attn[..., :kvl]
    if return_latent:
        return o_latent
    return torch.einsum("tnl,nvl->tnv", o_latent, w_uv)


def mla_latent_attention(q_latent, latent_cache, block_table, cu_seqlens_q, seqlens_kv,
                         scale, kv_lora_rank):
    """The kernel-sized piece of the absorbed path: MQA attention of
    q_latent (T, H, kvl+rope) over the latent pages, value = first kvl columns
    (auto_infer/layers/attention/mla.py:115-120)."""
    attn = paged_attention(q_latent, latent_cache, latent_cache, block_table,
                           cu_seqlens_q, seqlens_kv, scale)
    return attn[..., :kv_lora_rank]


def mla_nonabsorbed_attention(q_nope, q_pe, latent_tokens, kv_b_weight, num_heads,
                              qk_nope, v_head_dim, cu_seqlens, scale):
    """Non-absorbed form used to cross-check the absorbed algebra the way
    scripts/verify_mla_absorb.py:41-62 does: per-head K = [W_UK ckv | k_pe],
    V = W_UV ckv, dense causal attention over full sequences (q_len == kv_len)."""
    kvl = kv_b_weight.shape[-1]
    ckv, k_pe = latent_tokens[..., :kvl], latent_tokens[..., kvl:]
    kv = (ckv @ kv_b_weight.t()).view(-1, num_heads, qk_nope + v_head_dim)
    k_nope, v = kv.split([qk_nope, v_head_dim], dim=-1)
    k = torch.cat([k_nope, k_pe[:, None, :].expand(-1, num_heads, -1)], dim=-1)
    q = torch.cat([q_nope, q_pe], dim=-1)
    outs, start = [], 0
    for end in cu_seqlens:
        o, _ = _core_literal(q[start:end], k[start:end], v[start:end], scale)
        outs.append(o)
        start = end
    return torch.cat(outs, dim=0)


# --------------------------------------------------------------------------- #
# projection wrapper of the GQA family (adjacent to the path, used by the
# backend-level parity test)
# --------------------------------------------------------------------------- #
def rotate_half(x):
    """NeoX rotation (auto_infer/layers/rotary_embedding/__init__.py:10-12)."""
    x1, x2 = x.chunk(2, dim=-1)
    return torch.cat((-x2, x1), dim=-1)


def rms_norm(x, weight, eps):
    """Plain RMSNorm in fp32, cast back — stands in for the vendor op the
    reference calls (auto_infer/layers/norm.py:5-9)."""
    xf = x.float()
    return (xf * torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + eps)).to(x.dtype) * weight


def gqa_attention_block(x, w, prefix, n_q, n_kv, hd, scale, cos, sin, kv_cache, slots,
                        block_table, cu_seqlens_q, seqlens_kv, rms_eps=None):
    """The whole GQA attention sub-block as the reference wires it
    (auto_infer/layers/attention/gqa.py:27-49): packed QKV projection, optional
    per-head QK RMSNorm, NeoX RoPE, cache write BEFORE attention, paged
    attention, o_proj.  kv_cache (2, num_blocks, bs, Hkv, D).  Mutates the cache."""
    t = x.shape[0]
    p = prefix + "self_attn."
    qkv = x @ w[p + "qkv_proj.weight"].t()
    if w.get(p + "qkv_proj.bias") is not None:
        qkv = qkv + w[p + "qkv_proj.bias"]
    q, k, v = qkv.split((n_q * hd, n_kv * hd, n_kv * hd), dim=-1)
    q, k, v = q.view(t, n_q, hd), k.view(t, n_kv, hd), v.view(t, n_kv, hd)
    if w.get(p + "q_norm.weight") is not None:
        q = rms_norm(q, w[p + "q_norm.weight"], rms_eps)
        k = rms_norm(k, w[p + "k_norm.weight"], rms_eps)
    q = q * cos + rotate_half(q) * sin
    k = k * cos + rotate_half(k) * sin
    write_kv(k, v, kv_cache[0], kv_cache[1], slots)
    o = paged_attention(q, kv_cache[0], kv_cache[1], block_table, cu_seqlens_q, seqlens_kv, scale)
    return o.reshape(t, n_q * hd) @ w[p + "o_proj.weight"].t()


def ds_rope_interleave(x):
    """DeepSeek interleaved-rope regrouping
    (auto_infer/layers/rotary_embedding/__init__.py:15-23)."""
    d = x.shape[-1]
    return x.view(*x.shape[:-1], d // 2, 2).transpose(-1, -2).reshape(*x.shape[:-1], d)


def mla_absorbed_block(x, w, prefix, *, num_heads, qk_nope, qk_rope, v_head_dim, kv_lora_rank,
                       q_lora_rank, rms_eps, cos, sin, latent_cache, slots, block_table,
                       cu_seqlens_q, seqlens_kv, softmax_scale):
    """The whole absorbed-MLA sub-block as auto_infer/layers/attention/mla.py:76-122
    wires it, with the latent cached once.  Mutates the cache."""
    t = x.shape[0]
    nh, nope, rope, vd, kvl = num_heads, qk_nope, qk_rope, v_head_dim, kv_lora_rank
    if q_lora_rank is None:
        q = x @ w[prefix + "self_attn.q_proj.weight"].t()
    else:
        q = rms_norm(x @ w[prefix + "self_attn.q_a_proj.weight"].t(),
                     w[prefix + "self_attn.q_a_layernorm.weight"], rms_eps)
        q = q @ w[prefix + "self_attn.q_b_proj.weight"].t()
    q = q.view(t, nh, nope + rope)
    q_nope, q_pe = q.split([nope, rope], dim=-1)
    ckv_full = x @ w[prefix + "self_attn.kv_a_proj_with_mqa.weight"].t()
    ckv, k_pe = ckv_full.split([kvl, rope], dim=-1)
    ckv = rms_norm(ckv, w[prefix + "self_attn.kv_a_layernorm.weight"], rms_eps)
    k_pe = k_pe.view(t, 1, rope)
    q_pe = ds_rope_interleave(q_pe)
    k_pe = ds_rope_interleave(k_pe)
    q_pe = q_pe * cos + rotate_half(q_pe) * sin
    k_pe = k_pe * cos + rotate_half(k_pe) * sin
    w_uk, w_uv = build_absorb_weights(w[prefix + "self_attn.kv_b_proj.weight"], nh, nope, vd, kvl)
    k_latent = torch.cat([ckv.unsqueeze(1), k_pe], dim=-1).contiguous()
    write_kv(k_latent, None, latent_cache, None, slots)
    o = mla_absorbed_attention(q_nope, q_pe, latent_cache, block_table, cu_seqlens_q, seqlens_kv,
                               softmax_scale, w_uk, w_uv)
    return o.reshape(t, nh * vd) @ w[prefix + "self_attn.o_proj.weight"].t()


def mla_paged_block(x, w, prefix, *, num_heads, qk_nope, qk_rope, v_head_dim, kv_lora_rank,
                    q_lora_rank, rms_eps, cos, sin, k_cache, v_cache, slots, block_table,
                    cu_seqlens_q, seqlens_kv, softmax_scale, return_qkv=False):
    """The whole non-absorbed MLA sub-block as auto_infer/layers/attention/mla.py:134-164
    (and mla_paged, :23-64) wires it: per-head K = [k_nope | k_pe] and V written to caches of
    shape (num_blocks, bs, H, qk) / (num_blocks, bs, H, vd), multi-head paged attention with
    one kv head per query head, o_proj.  Mutates the caches."""
    t = x.shape[0]
    nh, nope, rope, vd = num_heads, qk_nope, qk_rope, v_head_dim
    if q_lora_rank is None:
        q = x @ w[prefix + "self_attn.q_proj.weight"].t()
    else:
        q = rms_norm(x @ w[prefix + "self_attn.q_a_proj.weight"].t(),
                     w[prefix + "self_attn.q_a_layernorm.weight"], rms_eps)
        q = q @ w[prefix + "self_attn.q_b_proj.weight"].t()
    q = q.view(t, nh, nope + rope)
    q_nope, q_pe = q.split([nope, rope], dim=-1)
    ckv = x @ w[prefix + "self_attn.kv_a_proj_with_mqa.weight"].t()
    ckv, k_pe = ckv.split([kv_lora_rank, rope], dim=-1)
    k_pe = k_pe.view(t, 1, rope)
    kv = rms_norm(ckv, w[prefix + "self_attn.kv_a_layernorm.weight"], rms_eps)
    kv = (kv @ w[prefix + "self_attn.kv_b_proj.weight"].t()).view(t, nh, nope + vd)
    k_nope, v = kv.split([nope, vd], dim=-1)
    q_pe = ds_rope_interleave(q_pe)
    k_pe = ds_rope_interleave(k_pe)
    q_pe = q_pe * cos + rotate_half(q_pe) * sin
    k_pe = k_pe * cos + rotate_half(k_pe) * sin
    q = torch.cat([q_nope, q_pe], dim=-1)
    k = torch.cat([k_nope, k_pe.expand(t, nh, rope)], dim=-1).contiguous()
    v = v.contiguous()
    write_kv(k, v, k_cache, v_cache, slots)
    o = paged_attention(q, k_cache, v_cache, block_table, cu_seqlens_q, seqlens_kv, softmax_scale)
    out = o.reshape(t, nh * vd) @ w[prefix + "self_attn.o_proj.weight"].t()
    return (out, q, k, v, o) if return_qkv else out


def softmax_scale_default(head_dim):
    return 1.0 / math.sqrt(head_dim)


# --------------------------------------------------------------------------- #
# 8-bit paged cache (no counterpart in the reference; from the definition, in 64 bits)
# --------------------------------------------------------------------------- #
def e4m3_round(x):
    """Nearest e4m3 value of ``x`` (float64), ties to even: 4 significant bits from 2^-6 up, steps
    of 2^-9 below, magnitudes past 448 (and infinities, NaN) become NaN."""
    x = x.double()
    e = torch.frexp(x.abs().clamp_min(2.0 ** -6)).exponent - 1
    step = torch.ldexp(torch.ones_like(x), e - 3)
    y = torch.round(x / step) * step
    return torch.where(y.abs() <= 448.0, y, torch.full_like(y, math.nan))


def fp8_scale_of(top):
    """Smallest power of two s >= 2^-126 with top <= 448 s."""
    s = 2.0 ** -126
    while top > 448.0 * s:
        s *= 2.0
    return s


def write_kv_fp8(rows, cache, scale, slots):
    """One of K / V: ``rows`` (T, Hkv, D) into ``cache`` (num_blocks, block_size, Hkv, D) holding the
    codes' values in float64, ``scale`` (num_blocks, Hkv) in float64; both updated in place.
    Later rows win when slots repeat; negative slots and slots past the pool are skipped."""
    num_blocks, bs, n_kv, _ = cache.shape
    by_page = {}
    for t, slot in enumerate(slots):
        if 0 <= slot < num_blocks * bs:
            by_page.setdefault(slot // bs, {})[slot % bs] = t
    for page, taken in by_page.items():
        for h in range(n_kv):
            x = rows[list(taken.values()), h].double()
            finite = x[torch.isfinite(x)].abs()
            call = fp8_scale_of(float(finite.max()) if finite.numel() else 0.0)
            old = float(scale[page, h])
            anew = 0 in taken or not (0.0 < old < math.inf)
            s = call if anew else max(old, call)
            if not anew and s > old:
                cache[page, :, h] = e4m3_round(cache[page, :, h] * (old / s))
            cache[page, list(taken), h] = e4m3_round(x / s)
            scale[page, h] = s
