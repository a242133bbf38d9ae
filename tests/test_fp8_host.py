"""8-bit cache: what the host refuses (no GPU needed; nothing is launched), and the oracle's rounding."""
import math
from types import SimpleNamespace

import pytest
import torch

from tests.fp8_cache import E4M3, empty_pool, orc


@pytest.fixture(scope="module")
def lib():
    from auto_infer_b200 import _lib, build
    build.build()
    return _lib.load()


def test_oracle_rounding_agrees_with_the_type():
    x = torch.cat([torch.linspace(-448, 448, 4001, dtype=torch.float64),
                   torch.exp2(torch.linspace(-12, 9, 1000, dtype=torch.float64)),
                   torch.arange(0, 256, dtype=torch.uint8).view(E4M3).double().nan_to_num(nan=0.0)])
    x = x[x.abs() <= 448].float()
    assert torch.equal(orc.e4m3_round(x), x.to(E4M3).double())
    assert orc.e4m3_round(torch.tensor([math.inf, -math.inf, math.nan, 500.0])).isnan().all()
    for top, s in ((448.0, 1.0), (449.0, 2.0), (1.75, 2.0 ** -8), (1.7500001, 2.0 ** -7), (0.0, 2.0 ** -126)):
        assert orc.fp8_scale_of(top) == s


def _write_args(**change):
    a = dict(key=1 << 20, key_stride=256, value=1 << 21, value_stride=256, key_cache=1 << 22, value_cache=1 << 23,
             key_scale=1 << 24, value_scale=1 << 25, slot_mapping=1 << 26, num_tokens=0, num_kv_heads=2, head_dim=128,
             block_size=16, num_blocks=4, status=None, stream=None)
    a.update(change)
    return list(a.values())


@pytest.mark.parametrize("change, code", [
    (dict(key_cache=None), -1), (dict(value_scale=None), -1), (dict(num_blocks=0), -1), (dict(num_kv_heads=0), -1),
    (dict(num_tokens=-1), -1), (dict(num_tokens=3, slot_mapping=None), -1), (dict(num_tokens=3, key_stride=255), -1),
    (dict(head_dim=64), -2), (dict(block_size=8), -2), (dict(block_size=24), -2), (dict(block_size=2048), -2),
    (dict(key_cache=(1 << 22) + 8), -3), (dict(num_tokens=3, key=(1 << 20) + 8), -3),
    (dict(num_tokens=3, value_stride=260), -3), (dict(block_size=1024, num_blocks=1 << 21), -5),
])
def test_slot_write_refusals(lib, change, code):
    assert lib.b200_reshape_and_cache_fp8(*_write_args(**change)) == code
    assert b"reshape_and_cache_fp8" in lib.b200_last_error()


def test_empty_write_launches_nothing(lib):
    assert lib.b200_reshape_and_cache_fp8(*_write_args()) == 0


def test_operators_refuse_cpu_tensors_and_unfit_caches():
    from auto_infer_b200 import ops
    kc, ks = empty_pool(2, 16, 2)
    rows = torch.zeros(3, 2, 128, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.reshape_and_cache_fp8(rows, rows, kc, kc, ks, ks, torch.zeros(3, dtype=torch.int32))
    assert ops._check_fp8_cache(kc, kc, ks, ks) == (2, 16, 2, 128)
    for bad in ((kc.float(), kc, ks, ks), (kc, kc[:1], ks, ks), (kc, kc, ks.double(), ks), (kc, kc, ks[:, :1], ks),
                (kc[:, ::2], kc[:, ::2], ks, ks), (kc[0], kc[0], ks, ks)):
        with pytest.raises(ValueError):
            ops._check_fp8_cache(*bad)


def _decode_args(**change):
    from auto_infer_b200._lib import DecodePlanInfo
    import ctypes
    info = DecodePlanInfo(num_ctas=4, num_items=1, num_partials=1)
    a = dict(q=1 << 20, q_stride=1024, key_cache=1 << 22, value_cache=1 << 23, key_scale=1 << 24, value_scale=1 << 25,
             num_blocks=4, block_size=16, block_table=1 << 26, bt_stride=4, table_rows=1, table_cols=4, plan=1 << 27,
             info=ctypes.byref(info), num_ctas=4, num_tokens=1, num_q_heads=8, num_kv_heads=2, head_dim=128, scale=0.1,
             workspace=1 << 28, workspace_bytes=1 << 16, out=1 << 29, out_is_f32=0, lse_out=None, status=None, stream=None)
    a.update(change)
    return list(a.values())


@pytest.mark.parametrize("change, code", [
    (dict(q=None), -1), (dict(block_table=None), -1), (dict(plan=None), -1), (dict(workspace=None), -1), (dict(out=None), -1),
    (dict(key_scale=None), -1), (dict(num_q_heads=7), -1), (dict(num_tokens=-1), -1), (dict(table_rows=0), -1),
    (dict(table_cols=0), -1), (dict(info=None, num_ctas=0), -1), (dict(head_dim=96), -2), (dict(block_size=8), -2),
    (dict(q=(1 << 20) + 4), -3), (dict(q_stride=1022), -3), (dict(out=(1 << 29) + 8), -3), (dict(plan=(1 << 27) + 4), -3),
    (dict(workspace_bytes=100), -6),
])
def test_decode_refusals(lib, change, code):
    assert lib.b200_paged_decode_gqa_fp8(*_decode_args(**change)) == code
    assert b"paged_decode_gqa_fp8" in lib.b200_last_error()


@pytest.mark.parametrize("change, code", [
    (dict(q=None), -1), (dict(block_table=None), -1), (dict(plan=None), -1), (dict(out=None), -1), (dict(value_scale=None), -1),
    (dict(num_q_heads=7), -1), (dict(num_tokens=-1), -1), (dict(max_ctas=-1), -1), (dict(table_cols=0), -1),
    (dict(head_dim=256), -2), (dict(block_size=8), -2), (dict(q=(1 << 20) + 8), -3), (dict(q_stride=1028), -3),
    (dict(out=(1 << 29) + 8), -3), (dict(plan=(1 << 27) + 4), -3), (dict(workspace=8), -3),
])
def test_prefill_refusals(lib, change, code):
    from auto_infer_b200._lib import PrefillPlanInfo
    import ctypes
    info = PrefillPlanInfo(num_items=1, num_tokens=1)
    a = dict(q=1 << 20, q_stride=1024, key_cache=1 << 22, value_cache=1 << 23, key_scale=1 << 24, value_scale=1 << 25,
             num_blocks=4, block_size=16, block_table=1 << 26, bt_stride=4, table_rows=1, table_cols=4, plan=1 << 27,
             info=ctypes.byref(info), max_ctas=0, num_tokens=1, num_q_heads=8, num_kv_heads=2, head_dim=128, scale=0.1,
             workspace=None, workspace_bytes=0, out=1 << 29, out_is_f32=0, lse_out=None, status=None, stream=None)
    a.update(change)
    assert lib.b200_paged_prefill_gqa_fp8(*a.values()) == code
    assert b"paged_prefill_gqa_fp8" in lib.b200_last_error()


def _model(**more):
    cfg = SimpleNamespace(head_dim=128, num_layers=3, rms_eps=1e-6)
    model = SimpleNamespace(cfg=cfg, n_q_local=8, n_kv_local=2, w={}, layer_prefix=lambda i: f"model.layers.{i}.",
                            device="cpu", dtype=torch.bfloat16, ATTENTION_FAMILY="gqa", _gqa_b200_kv_dtype=E4M3)
    model.__dict__.update(more)
    return model


def test_a_model_that_asks_for_8_bit_caches_gets_their_backend():
    from auto_infer_b200 import gqa, registry
    for mode, cls, base in (("paged", gqa.B200Fp8GqaBackend, gqa.B200GqaBackend),
                            ("graph", gqa.B200GraphFp8GqaBackend, gqa.B200GraphGqaBackend)):
        backend, caches = registry.build_attention_backend(_model(), mode, 5, 64)
        assert type(backend) is cls and isinstance(backend, base) and len(caches) == 3
        for k, v, ks, vs in caches:
            assert k.shape == v.shape == (5, 64, 2, 128) and k.dtype == v.dtype == E4M3
            assert ks.shape == vs.shape == (5, 2) and ks.dtype == vs.dtype == torch.float32
            assert not ks.any() and not vs.any() and k.data_ptr() != v.data_ptr()
        backend, caches = registry.build_mtp_attention_backend(_model(), mode, "model.mtp_layers.0.", 2, 16)
        assert type(backend) is cls and backend.num_layers == 1 and len(caches) == 1
        assert type(registry.build_attention_backend(_model(_gqa_b200_kv_dtype=torch.bfloat16), mode, 2, 16)[0]) is base
    with pytest.raises(ValueError, match="unsupported _gqa_b200_kv_dtype"):
        registry.build_attention_backend(_model(_gqa_b200_kv_dtype=torch.float16), "paged", 2, 16)
    with pytest.raises(NotImplementedError):
        registry.build_attention_backend(_model(), "dense")
    with pytest.raises(NotImplementedError, match="heads of 128"):
        registry.build_attention_backend(_model(cfg=SimpleNamespace(head_dim=64, num_layers=1, rms_eps=1e-6)), "paged", 2, 16)
    for bs in (8, 24, 2048):
        with pytest.raises(ValueError, match="power of two"):
            registry.build_attention_backend(_model(), "paged", 2, bs)


def test_prologue_without_a_cache_needs_somewhere_to_put_the_keys(lib):
    from auto_infer_b200 import ops
    x = torch.zeros(1, 2, 128, dtype=torch.bfloat16)
    cs = torch.zeros(1, 1, 128, dtype=torch.bfloat16)
    slots = torch.zeros(1, dtype=torch.int32)
    for kc, vc, sl, want_k in ((None, None, None, False), (x, None, slots, True), (None, None, slots, True), (x, x, None, True)):
        with pytest.raises(ValueError, match="go together"):
            ops.gqa_rope_cache(x, x, x, cs, cs, kc, vc, sl, want_k=want_k)
    a = dict(q=1 << 20, q_stride=256, k=1 << 20, k_stride=256, v=1 << 20, v_stride=256, cos=1 << 20, sin=1 << 20, cs=128,
             qn=None, kn=None, eps=1e-6, q_out=1 << 20, q_out_stride=256, k_out=None, key_cache=None, value_cache=None,
             slots=None, t=1, n_q=2, n_kv=2, d=128, block_size=0, num_blocks=0, status=None, stream=None)
    for change in (dict(), dict(k_out=1 << 20, slots=1 << 20), dict(k_out=1 << 20, key_cache=1 << 20),
                   dict(k_out=1 << 20, key_cache=1 << 20, value_cache=1 << 20, slots=1 << 20)):
        assert lib.b200_gqa_rope_cache(*(a | change).values()) == -1


def test_page_copy_refuses_what_is_not_words(lib):
    a = dict(src=1 << 20, dst=1 << 21, src_ids=1 << 22, dst_ids=None, num_ids=2, page_bytes=12, src_blocks=4, dst_blocks=4,
             status=None, stream=None)
    for change in (dict(page_bytes=6), dict(src=(1 << 20) + 2), dict(dst=(1 << 21) + 1)):
        assert lib.b200_copy_blocks(*(a | change).values()) == -3


def _block(entry, args):
    """The argument block of ``b200_call_fp8``: 8 bytes an argument, `scale` as a double."""
    import ctypes
    import struct
    from auto_infer_b200._lib import SIGNATURES
    types = SIGNATURES[entry][1]
    assert len(types) == len(args)
    words = [ctypes.addressof(a._obj) if hasattr(a, "_obj") else 0 if a is None else a for a in args]
    return struct.pack("".join("d" if t is ctypes.c_float else "q" for t in types), *words)


def test_calls_in_one_block_reach_the_same_checks(lib):
    """Each refusal of the entry points comes back from the block form, and integers that do not fit are refused."""
    calls = ((0, "b200_reshape_and_cache_fp8", _write_args, (dict(key_cache=None), dict(head_dim=64), dict(block_size=24),
                                                             dict(num_tokens=3, key_stride=255), dict(num_tokens=0))),
             (1, "b200_paged_decode_gqa_fp8", _decode_args, (dict(q=None), dict(num_q_heads=7), dict(head_dim=96),
                                                             dict(q_stride=1022), dict(workspace_bytes=100),
                                                             dict(info=None, num_ctas=0))))
    for number, name, make, changes in calls:
        for change in changes:
            assert lib.b200_call_fp8(number, _block(name, make(**change))) == getattr(lib, name)(*make(**change))
            assert number == 0 or lib.b200_last_error()
        for field in ("num_blocks", "head_dim"):
            assert lib.b200_call_fp8(number, _block(name, make(**{field: 2 ** 32 + 128}))) == -1
            assert b"does not fit" in lib.b200_last_error()
    assert lib.b200_call_fp8(1, _block(calls[1][1], _decode_args(workspace_bytes=-1))) == -1
    assert lib.b200_call_fp8(3, b"\0" * 256) == -1 and b"unknown entry 3" in lib.b200_last_error()
    assert lib.b200_call_fp8(1, None) == -1


@pytest.mark.parametrize("cu, kv, n_kv, ctas", [
    ([5], [9000], 1, 148), ([5, 10, 15], [9000, 200, 40], 2, 148), ([40] * 3, [5000, 1, 0], 8, 148), ([2000], [2000], 1, 148),
    ([1, 2, 3], [100000, 70000, 3], 3, 20), ([16], [130], 1, 148), ([0], [50], 2, 4), ([3], [0], 2, 4), ([700], [40000], 1, 1)])
def test_a_cut_plan_covers_every_tile_once(lib, cu, kv, n_kv, ctas):
    """The pieces are the items' tiles, each once; records are dealt in the order of the tiles; nothing is a sliver."""
    import ctypes
    from auto_infer_b200._lib import PrefillPlanInfo
    n_q, n = 4 * n_kv, len(cu)
    ints = lambda x: (ctypes.c_int32 * len(x))(*x)
    size = lib.b200_prefill_plan_bytes(n, cu[-1], n_q, n_kv)
    size += lib.b200_prefill_split_bytes(size // 32, ctas)
    plan = torch.full((size // 4 + 8,), -7, dtype=torch.int32)
    info, partials = PrefillPlanInfo(), ctypes.c_int(-1)
    assert lib.b200_prefill_plan(ints(cu), ints(kv), None, n, n_q, n_kv, 0, plan.data_ptr(), size, ctypes.byref(info)) == 0
    before = plan[:info.plan_ints].clone()
    assert lib.b200_prefill_split(plan.data_ptr(), size, ctas, ctypes.byref(info), ctypes.byref(partials)) == 0
    items = before[16:16 + 8 * info.num_items].view(-1, 8)
    assert torch.equal(plan[16:16 + 8 * info.num_items].view(-1, 8), items) and (plan[info.plan_ints:] == -7).sum() >= 8
    pieces, at, groups_at, groups = plan[4:8].tolist()
    assert partials.value <= 2 * ctas and info.plan_ints * 4 <= size
    if pieces == 0:
        assert partials.value == 0 and torch.equal(plan[:info.plan_ints], before)
        return
    rows = plan[at:at + 12 * pieces].view(-1, 12)
    assert (rows[:-1, 3] >= rows[1:, 3]).all() and pieces <= info.num_items + ctas
    parts = {}
    for x in rows.tolist():
        parts.setdefault((x[0], x[1], x[2]), []).append((x[8], x[3], x[9]))
    seen = []
    for item in items.tolist():
        runs = sorted(parts.pop((item[0], item[1], item[2])))
        assert runs[0][0] == 0 and sum(r[1] for r in runs) == item[3]
        for a, b in zip(runs, runs[1:]):
            assert a[0] + a[1] == b[0] and b[2] == a[2] + 1 and min(a[1], b[1]) >= 4
        assert (runs[0][2] == -1) == (len(runs) == 1)
        if len(runs) > 1:
            seen.append([runs[0][2], len(runs), item[1], item[2], item[5], item[6]])
    assert not parts and groups == len(seen)
    assert plan[groups_at:groups_at + 8 * groups].view(-1, 8)[:, :6].tolist() == seen
    assert sum(s[1] for s in seen) == partials.value


def test_split_refusals(lib):
    import ctypes
    from auto_infer_b200._lib import PrefillPlanInfo
    plan, info, partials = torch.zeros(64, dtype=torch.int32), PrefillPlanInfo(), ctypes.c_int(0)
    args = [plan.data_ptr(), 256, 148, ctypes.byref(info), ctypes.byref(partials)]
    assert lib.b200_prefill_split(*args) == -1                               # not a plan
    assert lib.b200_prefill_plan(None, None, None, 0, 8, 2, 0, plan.data_ptr(), 256, ctypes.byref(info)) == 0
    assert lib.b200_prefill_split(*args) == -6                               # no room
    assert lib.b200_prefill_split(None, *args[1:]) == -1 and lib.b200_prefill_split(*args[:2], 0, *args[3:]) == -1
    assert lib.b200_prefill_split(*args[:2], 5000, *args[3:]) == -1
    assert lib.b200_prefill_split_bytes(-1, 4) == 0 and lib.b200_prefill_split_workspace_bytes(-1) == 0


def test_backends_over_different_caches_do_not_share_a_contexts_plans(monkeypatch):
    """A 16-bit and an 8-bit backend of one head geometry on one context: a plan for each, whichever comes first."""
    from auto_infer_b200 import metadata
    built = []

    class Plans:
        capacity_seqs = 16

        def __init__(self, *args, split_prefill=False, **kw):
            self.split_prefill = split_prefill
            built.append(self)

    monkeypatch.setattr(metadata, "StepMetadata", Plans)
    for order in ((2, 1), (1, 2)):
        built.clear()
        ctx, pools = SimpleNamespace(cu_seqlens_q=[3, 20], seqlens_kv=[50, 40]), {1: {}, 2: {}}
        got = {n: metadata.step_metadata(ctx, 8, 2, 128, "cpu", pool=pools[n], kv_elem_bytes=n) for n in order}
        assert got[1].split_prefill and not got[2].split_prefill and len(built) == 2
        for n in order:
            assert metadata.step_metadata(ctx, 8, 2, 128, "cpu", pool=pools[n], kv_elem_bytes=n) is got[n]
            assert metadata.cached_step_metadata(ctx, 8, 2, 128, "cpu", n) is got[n]
            assert list(pools[n].values()) == [got[n]]
        assert metadata.cached_step_metadata(ctx, 8, 2, 128, "cpu") is got[2]
        assert len(built) == 2


def _producer(name):
    """The loads of a kernel's producer and the waits it leaves by, as two pieces of source."""
    import os
    from auto_infer_b200 import build
    text = open(os.path.join(build.CSRC, name)).read()
    text = text[text.index("tma_prefetch_desc(&v_map)"):]
    loop, drain = text.split("// drain: ", 1)
    return loop, drain[:drain.index("return;" if "decode" in name else "} else if")]


@pytest.mark.parametrize("name, waits", [("paged_decode_gqa_fp8.cu", 1), ("paged_prefill_gqa_fp8.cu", 2)])
def test_a_producer_that_gives_up_loads_nothing_more_and_waits_for_what_it_has_loaded(name, waits):
    """Read from the source, as no wait of a sound kernel runs out: between a producer's wait for a free stage and the load
    into it stands the way out of the loop (a barrier is armed behind it, or by a lane that saw the stage free), and the
    waits before it leaves pass by no abort flag."""
    import re
    loop, drain = _producer(name)
    steps = re.findall(r"mbar_wait_\w+\(&sm\.\w*empty\[s\w?\]|__any_sync\(0xffffffffu, \*abort_flag\)\) break|"
                       r"!__all_sync\(0xffffffffu, stage_free\)\) break|stage_free\) mbar_arrive_expect_tx|"
                       r"mbar_arrive_expect_tx|tma_load_4d", loop)
    kinds = "".join("w" if "wait" in s else "b" if "break" in s else "a" if s.startswith("stage_free") else "l" for s in steps)
    assert re.fullmatch("(wa?bl+){%d}b?" % waits, kinds), kinds
    assert "mbar_wait_landed" in drain and "abort" not in drain and not re.search("mbar_wait_(bounded|limited)", drain)


def test_tensor_memory_is_not_given_back_under_matrix_products():
    """Each of the two issuing warps ends with a commit of its own and waits for it whatever the abort flag says."""
    import os
    import re
    from auto_infer_b200 import build
    text = open(os.path.join(build.CSRC, "paged_prefill_gqa_fp8.cu")).read()
    ends = [m.start() for m in re.finditer(r"umma_commit\(&sm\.mma_idle\[(\d)\]\);\s+mbar_wait_landed\(&sm\.mma_idle\[\1\], 0\);", text)]
    roles = [text.index(s) for s in ("} else if (warp == 9) {", "} else if (warp == 10) {", "} else if (warp < 8) {")]
    assert len(ends) == 2 and roles[0] < ends[0] < roles[1] < ends[1] < roles[2] < text.index("tmem_dealloc")
