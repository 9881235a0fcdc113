"""Attention weights, eviction and head-128 decode on the host (CPU, no kernel runs): what the C entry points refuse
before any device work, the workspace and split-count arithmetic, and what the Python operators check of their
arguments."""
import ctypes

import pytest
import torch

from vllm_quantpack_b200 import _lib
from vllm_quantpack_b200.attention import ops

F = ctypes.c_float
ONE = ctypes.c_void_p(16)      # a non-null, aligned stand-in for device pointers that a refused call never reads


@pytest.fixture(scope="module")
def lib():
    from vllm_quantpack_b200 import build
    build.build()
    return _lib.load()


def weights_rc(lib, **over):
    """qp_accumulate_attn_weights with arguments that pass every check, but those overridden."""
    a = dict(fmt=0, dtype=0, q=ONE, q_st=1024, q_sh=256, tokens=4, seqs=1, cu=ONE, used=ONE, max_q=4, max_k=100, bt=ONE,
             bt_st=8, cache=ONE, bs=16, block=16 * 4 * 264, head=16 * 264, slot=264, k=0, ks=128, v=132, vs=260, nq=4,
             nkv=4, hs=256, scale=F(0.0625), signs=ONE, rot=0, after=0, window=0, cap=F(0.0), lse=ONE, w=ONE, wb=64,
             wsl=1, wh=16, ws=ONE, nbytes=1 << 40, stream=None)
    assert set(over) <= set(a)
    a.update(over)
    return lib.qp_accumulate_attn_weights(*a.values()), lib.qp_last_error().decode()


@pytest.mark.parametrize("over,code,words", [
    (dict(fmt=2), 2, "format"), (dict(dtype=3), 2, "dtype"), (dict(hs=64), 2, "head size"),
    (dict(slot=272), 3, "contiguous"), (dict(ks=120), 3, "field"), (dict(bs=24), 3, "block size"),
    (dict(cache=ctypes.c_void_p(8)), 3, "16-byte"), (dict(nq=6), 1, "heads"), (dict(nkv=0), 1, "heads"),
    (dict(max_q=-1), 1, "sizes"), (dict(after=-1), 1, "tokens_after"), (dict(window=-2), 1, "window"),
    (dict(cap=F(-1.0)), 1, "softcap"), (dict(cap=F(float("nan"))), 1, "softcap"), (dict(lse=None), 1, "null"),
    (dict(w=None), 1, "null"), (dict(q=None), 1, "null"), (dict(nbytes=1000), 4, "workspace"),
    (dict(ws=ctypes.c_void_p(8)), 4, "workspace"), (dict(seqs=70000), 2, "large"),
    (dict(max_q=1 << 30), 2, "large"),
])
def test_weights_refuses(lib, over, code, words):
    rc, msg = weights_rc(lib, **over)
    assert rc == code and words in msg, (rc, msg)


@pytest.mark.parametrize("over", [dict(seqs=0), dict(tokens=0), dict(max_q=0), dict(max_k=0)])
def test_weights_of_nothing_is_no_work(lib, over):
    assert weights_rc(lib, **over)[0] == 0


def evict_rc(lib, **over):
    a = dict(cache=ONE, cell=264, bs=16, block=16 * 4 * 264, head=16 * 264, slot=264, nkv=4, w=ONE, wb=64, wsl=1, wh=16,
             seqs=1, used=ONE, max_k=100, bt=ONE, bt_st=8, obt=None, obt_st=0, keep=50, first=4, last=10, kept=ONE,
             out=ONE, ws=ONE, nbytes=1 << 40, stream=None)
    assert set(over) <= set(a)
    a.update(over)
    return lib.qp_evict_cache(*a.values()), lib.qp_last_error().decode()


@pytest.mark.parametrize("over,code,words", [
    (dict(keep=0), 1, "keep"), (dict(first=-1), 1, "keep"), (dict(last=-1), 1, "keep"), (dict(first=41), 1, "keep"),
    (dict(first=51, last=0), 1, "keep"), (dict(cell=260), 2, "cells"), (dict(cell=2048), 2, "cells"),
    (dict(slot=268), 3, "aligned"), (dict(cache=ctypes.c_void_p(4)), 3, "aligned"), (dict(nkv=0), 1, "sizes"),
    (dict(bs=0), 1, "sizes"), (dict(max_k=-1), 1, "sizes"), (dict(w=None), 1, "null"), (dict(kept=None), 1, "null"),
    (dict(used=None), 1, "null"), (dict(out=None), 1, "null"), (dict(nbytes=16), 4, "workspace"),
    (dict(seqs=70000), 2, "large"),
])
def test_evict_refuses(lib, over, code, words):
    rc, msg = evict_rc(lib, **over)
    assert rc == code and words in msg, (rc, msg)


def test_evict_of_nothing_is_no_work(lib):
    assert evict_rc(lib, seqs=0)[0] == 0


def test_workspace_sizes_cover_their_parts(lib):
    # one record of 32 rows x 256 channels in two fp16 terms per (sequence, KV head) when decoding
    assert lib.qp_attn_weights_workspace_bytes(8, 8, 1, 24, 4, 256) >= 8 * 4 * 16 * 256 * 4
    # a prompt's rows, all of them, at every head size
    for hs in (128, 256, 512):
        for tokens, seqs, longest in ((1000, 1, 1000), (1003, 3, 900), (5, 5, 1)):
            need = lib.qp_attn_weights_workspace_bytes(tokens, seqs, longest, 24, 4, hs)
            assert need >= tokens * 24 * hs * 4
    # one long prompt among many short requests does not make every request a long one
    assert lib.qp_attn_weights_workspace_bytes(4000, 64, 3937, 8, 8, 128) < 64 * 3937 * 8 * 128 * 4
    assert lib.qp_evict_workspace_bytes(3, 4, 1000, 256) >= 3 * 8 + 16 + 3 * 4 * 8 * 4


def test_head_128_split_counts(lib):
    """One partial where a sequence is no longer than a CTA's warps take at a time, bounded by the shares that can meet
    in it otherwise; the other head sizes as before."""
    assert lib.qp_decode_num_splits_head(128, 8, 4, 8, 200, 148) == 1
    one = lib.qp_decode_num_splits_head(128, 8, 1, 4, 131072, 148)
    assert 74 <= one <= 512
    assert 2 <= lib.qp_decode_num_splits_head(128, 16, 128, 8, 32768, 148) <= 5
    assert lib.qp_decode_num_splits_head(256, 8, 1, 4, 131072, 148) == lib.qp_decode_num_splits(1, 4, 131072, 148)


# ---------------------------------------------------------------- the Python operators


@pytest.fixture
def calls(monkeypatch):
    """ops with the library, the device check and the workspace replaced: records the C calls."""
    seen = []
    monkeypatch.setattr(ops._lib, "call", lambda name, *a: seen.append((name, a)))
    monkeypatch.setattr(ops, "_memo", lambda *a: 0)
    monkeypatch.setattr(ops, "workspace", lambda device, n: torch.empty(1024, dtype=torch.uint8))
    monkeypatch.setattr(ops, "_stream", lambda device: 0)
    monkeypatch.setattr(ops, "_check_device", lambda device, **t: None)
    monkeypatch.setattr(ops.rht, "device_sign_bits", lambda hs, device: torch.zeros(hs // 32, dtype=torch.int32))
    return seen


def cache_views(blocks=6, bs=16, nkv=2, hs=128):
    phs = hs // 2 + 4
    kv = torch.zeros((blocks, nkv, bs, 2 * phs), dtype=torch.uint8)
    base = torch.tensor([], dtype=torch.float32).set_(kv.untyped_storage())
    st = [s // 4 for s in kv.stride()]
    ks = torch.as_strided(base, (blocks, bs, nkv), (st[0], st[2], st[1]), hs // 2 // 4)
    vs = torch.as_strided(base, (blocks, bs, nkv), (st[0], st[2], st[1]), (phs + hs // 2) // 4)
    kc, vc = kv.transpose(1, 2).split(phs, dim=-1)
    return kc, vc, ks, vs


def weights_args(**over):
    kc, vc, ks, vs = cache_views()
    a = dict(q=torch.zeros((3, 4, 128), dtype=torch.bfloat16), key_cache=kc, value_cache=vc,
             weights=ops.new_attention_weights(ks), lse=torch.zeros((3, 4)),
             cu_seqlens_q=torch.tensor([0, 1, 3], dtype=torch.int32), max_seqlen_q=2,
             seqused_k=torch.tensor([5, 9], dtype=torch.int32), max_seqlen_k=9, softmax_scale=0.1,
             block_table=torch.zeros((2, 1), dtype=torch.int32), k_scale_cache=ks, v_scale_cache=vs)
    a.update(over)
    return a


def test_weights_call(calls):
    a = weights_args()
    assert a["weights"].shape == (6, 16, 2) and a["weights"].stride() == (32, 1, 16)
    assert ops.accumulate_attention_weights(**a) is a["weights"]
    name, args = calls[0]
    assert name == "qp_accumulate_attn_weights" and len(args) == len(_lib.SIGNATURES[name][1])


@pytest.mark.parametrize("over,error,words", [
    (dict(weights=torch.zeros((6, 2, 16))), ValueError, "weights"),
    (dict(weights=torch.zeros((6, 16, 2), dtype=torch.float64)), ValueError, "weights"),
    (dict(lse=torch.zeros((3, 5))), ValueError, "lse"),
    (dict(lse=torch.zeros((4, 3)).T), ValueError, "lse"),
    (dict(lse=torch.zeros((3, 4), dtype=torch.float16)), ValueError, "lse"),
    (dict(seqused_k=torch.tensor([5, 9])), TypeError, "seqused_k"),
    (dict(block_table=torch.zeros((2, 2), dtype=torch.int32)[:, ::2]), ValueError, "block_table"),
    (dict(q=torch.zeros((3, 128, 4), dtype=torch.bfloat16).transpose(1, 2)), ValueError, "contiguous"),
    (dict(q=torch.zeros((3, 4, 128))), TypeError, "dtype"),
])
def test_weights_argument_checks(calls, over, error, words):
    with pytest.raises(error, match=words):
        ops.accumulate_attention_weights(**weights_args(**over))
    assert not calls


def evict_args(**over):
    kc, vc, ks, vs = cache_views()
    a = dict(key_cache=kc, value_cache=vc, weights=ops.new_attention_weights(ks),
             seqused_k=torch.tensor([40, 9], dtype=torch.int32), max_seqlen_k=40,
             block_table=torch.zeros((2, 3), dtype=torch.int32), keep=20, keep_first=2, keep_last=4, k_scale_cache=ks,
             v_scale_cache=vs)
    a.update(over)
    return a


def test_evict_call(calls):
    kept, new = ops.evict_cache(**evict_args())
    assert kept.shape == (2, 2, 20) and kept.dtype == torch.int32 and new.shape == (2,)
    name, args = calls[0]
    assert name == "qp_evict_cache" and len(args) == len(_lib.SIGNATURES[name][1])
    assert args[1] == 136       # the cell of an int4 head-128 cache, from the views
    used = torch.tensor([40, 9], dtype=torch.int32)
    assert ops.evict_cache(**evict_args(seqused_k=used, seqused_out=used))[1] is used


@pytest.mark.parametrize("over,error,words", [
    (dict(weights=torch.zeros((6, 2, 16))), ValueError, "weights"),
    (dict(seqused_k=torch.tensor([40, 9])), TypeError, "seqused_k"),
    (dict(block_table=torch.zeros((1, 3), dtype=torch.int32)), ValueError, "block_table"),
    (dict(out_block_table=torch.zeros((2, 1), dtype=torch.int32)), ValueError, "out_block_table"),
    (dict(out_block_table=torch.zeros((1, 2), dtype=torch.int32)), ValueError, "out_block_table"),
    (dict(out_block_table=torch.zeros((2, 2))), TypeError, "out_block_table"),
    (dict(seqused_out=torch.zeros(2)), ValueError, "seqused_out"),
    (dict(seqused_out=torch.zeros(3, dtype=torch.int32)), ValueError, "seqused_out"),
])
def test_evict_argument_checks(calls, over, error, words):
    with pytest.raises(error, match=words):
        ops.evict_cache(**evict_args(**over))
    assert not calls


def test_lse_output_argument_checks(calls):
    kc, vc, ks, vs = cache_views()
    q = torch.zeros((2, 4, 128), dtype=torch.bfloat16)
    a = dict(cu_seqlens_q=torch.tensor([0, 2], dtype=torch.int32), max_seqlen_q=2,
             seqused_k=torch.tensor([5], dtype=torch.int32), max_seqlen_k=5, softmax_scale=0.1,
             block_table=torch.zeros((1, 1), dtype=torch.int32), k_scale_cache=ks, v_scale_cache=vs, num_splits=1)
    lse = torch.zeros((2, 4))
    ops.paged_decode(q, kc, vc, torch.empty_like(q), lse_out=lse, **a)
    assert len(calls) == 1 and lse.data_ptr() in calls[0][1]
    with pytest.raises(ValueError, match="lse_out"):
        ops.paged_decode(q, kc, vc, torch.empty_like(q), lse_out=torch.zeros((4, 2)), **a)
    with pytest.raises(ValueError, match="lse_out"):
        ops.paged_decode(q, kc, vc, torch.empty((2, 4, 128)), lse_out=lse, out_fp32_lse=torch.zeros((2, 4)), **a)
    with pytest.raises(ValueError, match="lse_out"):
        ops.paged_decode(q, kc, vc, torch.empty_like(q), lse_out=lse, partials_only=True, **a)
    assert len(calls) == 1


def decode_args(**over):
    """paged_decode of two sequences over a cache of head 128."""
    kc, vc, ks, vs = cache_views()
    q = torch.zeros((3, 4, 128), dtype=torch.bfloat16)
    a = dict(q=q, key_cache=kc, value_cache=vc, out=torch.empty_like(q),
             cu_seqlens_q=torch.tensor([0, 1, 3], dtype=torch.int32), max_seqlen_q=2,
             seqused_k=torch.tensor([5, 9], dtype=torch.int32), max_seqlen_k=9, softmax_scale=0.1,
             block_table=torch.zeros((2, 1), dtype=torch.int32), k_scale_cache=ks, v_scale_cache=vs, num_splits=1)
    a.update(over)
    return a


def test_decode_takes_a_table_of_one_dimension(calls):
    """One request's block table as a row, without the sequence axis; for several requests it is refused."""
    table = torch.arange(4, dtype=torch.int32)
    one = dict(q=torch.zeros((1, 4, 128), dtype=torch.bfloat16), out=torch.zeros((1, 4, 128), dtype=torch.bfloat16),
               cu_seqlens_q=torch.tensor([0, 1], dtype=torch.int32), seqused_k=torch.tensor([5], dtype=torch.int32))
    ops.paged_decode(**decode_args(block_table=table, **one))
    ops.paged_decode(**decode_args(block_table=table[None], **one))
    (name, flat), (_, rows) = calls
    assert name == "qp_paged_decode" and table.data_ptr() in flat and len(flat) == len(_lib.SIGNATURES[name][1])
    at = flat.index(table.data_ptr())
    assert flat[at + 1] == 1 and rows[at + 1] == 4     # the row stride, which one sequence does not use
    with pytest.raises(ValueError, match="block_table"):
        ops.paged_decode(**decode_args(block_table=table))
    assert len(calls) == 2


@pytest.mark.parametrize("name", ["cu_seqlens_q", "seqused_k", "block_table"])
def test_decode_names_the_wrong_index_tensor(calls, name):
    a = decode_args()
    with pytest.raises(TypeError, match=f"^{name} "):
        ops.paged_decode(**dict(a, **{name: a[name].long()}))
    wide = torch.zeros((*a[name].shape[:-1], 2 * 3), dtype=torch.int32)[..., ::2]
    with pytest.raises(ValueError, match=f"^{name} "):
        ops.paged_decode(**dict(a, **{name: wide}))
    assert not calls


# ---------------------------------------------------------------- tensors on another device


class On:
    """A tensor on a device, as far as the check looks."""

    def __init__(self, index):
        self.device = torch.device("cuda", index) if index >= 0 else torch.device("cpu")

    def get_device(self):
        return -1 if self.device.index is None else self.device.index


def test_device_check(monkeypatch):
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)
    here = torch.device("cuda", 1)
    ops._check_device(here, out=On(1), lse_out=None)
    for wrong in (On(0), On(-1)):
        with pytest.raises(ValueError, match="lse_out"):
            ops._check_device(here, out=On(1), lse_out=wrong)
    for elsewhere in (torch.device("cuda", 0), torch.device("cpu")):
        with pytest.raises(ValueError, match="current device"):
            ops._check_device(elsewhere, out=On(1))


@pytest.mark.parametrize("hs", [128, 256])
def test_every_tensor_a_kernel_gets_is_checked(calls, monkeypatch, hs):
    """Each tensor whose address goes to a launch goes through the device check first, at every head size."""
    seen = {}
    monkeypatch.setattr(ops, "_check_device", lambda device, **t: seen.update(
        {id(x): device for x in t.values() if x is not None}))
    kc, vc, ks, vs = cache_views(hs=hs)
    q, out = (torch.zeros((3, 4, hs), dtype=torch.bfloat16) for _ in range(2))
    cu, used = torch.tensor([0, 1, 3], dtype=torch.int32), torch.tensor([5, 9], dtype=torch.int32)
    table, lse, sinks = torch.zeros((2, 1), dtype=torch.int32), torch.zeros((3, 4)), torch.zeros(4)
    ws, out32 = torch.empty(64, dtype=torch.uint8), torch.zeros((3, 4, hs))
    weights = ops.new_attention_weights(ks)
    common = dict(softmax_scale=0.1, k_scale_cache=ks, v_scale_cache=vs, ws=ws)
    index = dict(cu_seqlens_q=cu, seqused_k=used, max_seqlen_k=9, block_table=table)
    monkeypatch.setattr(ops._lib, "load", lambda: type("L", (), {
        "qp_prefill_workspace_bytes": lambda *a: 0, "qp_prefill_varlen_workspace_bytes": lambda *a: 0})())
    for fn, given, kw in [
            (ops.paged_decode, [out, lse, sinks], dict(max_seqlen_q=2, sinks=sinks, lse_out=lse, num_splits=1, **index)),
            (ops.paged_decode, [out32, lse], dict(max_seqlen_q=2, out_fp32_lse=lse, num_splits=1, **index)),
            (ops.prefill_varlen, [out, lse, sinks], dict(sinks=sinks, lse_out=lse, **index)),
            (ops.prefill_varlen, [out32, lse], dict(out_fp32_lse=lse, **index)),
            (ops.prefill, [out, lse], dict(block_row=table[0], n=9, lse_out=lse)),
            (ops.prefill, [out32, lse], dict(block_row=table[0], n=9, out_fp32_lse=lse))]:
        seen.clear()
        fn(q, kc, vc, given[0], **kw, **common)
        wanted = given + [kc, ws] + [t for t in kw.values() if isinstance(t, torch.Tensor)]
        assert all(id(t) in seen for t in wanted), fn.__name__
        assert set(seen.values()) == {q.device}
    seen.clear()
    ops.accumulate_attention_weights(q, kc, vc, weights, lse=lse, max_seqlen_q=2, **index, **common)
    assert all(id(t) in seen for t in (kc, weights, lse, cu, used, table, ws))
    seen.clear()
    ops.evict_cache(kc, vc, weights, seqused_k=used, max_seqlen_k=9, block_table=table, out_block_table=table.clone(),
                    keep=5, k_scale_cache=ks, v_scale_cache=vs, ws=ws)
    assert all(id(t) in seen for t in (weights, used, table, ws))


@pytest.mark.parametrize("hs", [128, 256, 512])
def test_host_tensors_are_refused(monkeypatch, hs):
    """Nothing on the host reaches a launch."""
    monkeypatch.setattr(ops._lib, "call", lambda *a: pytest.fail("a launch"))
    kc, vc, ks, vs = cache_views(hs=hs)
    q = torch.zeros((3, 4, hs), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="cpu"):
        ops.paged_decode(q, kc, vc, torch.empty_like(q), cu_seqlens_q=torch.tensor([0, 1, 3], dtype=torch.int32),
                         max_seqlen_q=2, seqused_k=torch.tensor([5, 9], dtype=torch.int32), max_seqlen_k=9,
                         softmax_scale=0.1, block_table=torch.zeros((2, 1), dtype=torch.int32), k_scale_cache=ks,
                         v_scale_cache=vs, num_splits=1, ws=torch.empty(64, dtype=torch.uint8))


# ---------------------------------------------------------------- tables and lengths that are too short


@pytest.mark.parametrize("over,words", [
    (dict(max_seqlen_k=17), "block_table"),                                                # two pages, one in the table
    (dict(block_table=torch.zeros((1, 1), dtype=torch.int32)), "block_table"),             # a row short
    (dict(seqused_k=torch.tensor([5], dtype=torch.int32)), "seqused_k"),                   # a length short
    (dict(block_table=torch.zeros(4, dtype=torch.int32)), "block_table"),                  # one row for two sequences
])
def test_weights_refuse_short_tables(calls, over, words):
    with pytest.raises(ValueError, match=words):
        ops.accumulate_attention_weights(**weights_args(**over))
    assert not calls


@pytest.mark.parametrize("over", [
    dict(max_seqlen_k=49),                                                                 # four pages, three in the table
    dict(block_table=torch.zeros((2, 2), dtype=torch.int32)),
    dict(block_table=torch.zeros(6, dtype=torch.int32)),
])
def test_evict_refuses_short_tables(calls, over):
    """In place a table row is written through as far as the lengths and the budget go."""
    with pytest.raises(ValueError, match="^block_table"):
        ops.evict_cache(**evict_args(**over))
    assert not calls


def test_tables_that_just_fit(calls):
    ops.accumulate_attention_weights(**weights_args(max_seqlen_k=16))
    ops.evict_cache(**evict_args(max_seqlen_k=48))
    one = dict(seqused_k=torch.tensor([40], dtype=torch.int32), block_table=torch.zeros(3, dtype=torch.int32))
    ops.evict_cache(**evict_args(**one))                          # one sequence's row
    ops.evict_cache(**evict_args(out_block_table=torch.zeros(2, dtype=torch.int32), **one))
    ops.evict_cache(**evict_args(out_block_table=torch.zeros((2, 2), dtype=torch.int32)))   # 20 of 40 tokens stay
    with pytest.raises(ValueError, match="^out_block_table"):
        ops.evict_cache(**evict_args(out_block_table=torch.zeros(1, dtype=torch.int32), **one))
    assert len(calls) == 5


# ---------------------------------------------------------------- workspaces


def test_workspaces_of_streams(monkeypatch):
    """Eager calls on two streams get two buffers; captured ones, and those on the default stream, the device's own."""
    monkeypatch.setattr(ops, "_workspaces", {})
    monkeypatch.setattr(ops, "_retired", [])
    now = dict(stream=0, capturing=False)
    monkeypatch.setattr(ops, "_stream", lambda device: now["stream"])
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: now["capturing"])

    def get(stream, nbytes=100, capturing=False):
        now.update(stream=stream, capturing=capturing)
        return ops.workspace("cpu", nbytes)

    own = get(0)
    a, b = get(7), get(9)
    assert len({t.data_ptr() for t in (own, a, b)}) == 3
    assert get(7) is a and get(9) is b and get(0) is own
    assert get(7, capturing=True) is own and get(11, capturing=True) is own
    now.update(stream=7, capturing=False)
    big = ops.reserve_workspace("cpu", 3 << 20)        # grown for a capture to come, from whatever stream
    assert big.numel() >= 3 << 20 and get(13, 3 << 20, capturing=True) is big and get(0) is big
    assert get(7) is a
    assert any(t is own for t in ops._retired)         # a graph may hold the smaller one


def test_workspace_reserved_at_start(monkeypatch):
    """The metadata builder's reservation covers captured steps and eager ones on its stream."""
    from vllm_quantpack_b200.attention import int4_kv
    seen = []
    monkeypatch.setattr(ops, "reserve_workspace", lambda device, n: seen.append(("own", device, n)))
    monkeypatch.setattr(ops, "workspace", lambda device, n: seen.append(("stream", device, n)))
    monkeypatch.setattr(ops, "sm_count", lambda device: 148)
    monkeypatch.setattr(int4_kv, "decode_workspace_bound", lambda *a: 12345)
    model = type("M", (), dict(get_num_attention_heads=lambda s, p: 24, get_num_kv_heads=lambda s, p: 4,
                               get_head_size=lambda s: 256, max_model_len=4096))()
    config = type("C", (), dict(model_config=model, parallel_config=None))()
    int4_kv.reserve_decode_workspace(type("B", (), dict(seq_threshold_3D=16))(), config, "cuda:0")
    assert seen == [("own", "cuda:0", 12345), ("stream", "cuda:0", 12345)]
