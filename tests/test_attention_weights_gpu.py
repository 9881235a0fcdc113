"""Accumulated attention weights (csrc/qp_weights.cu) against the definition in fp64 from the same cache bytes: both
formats, head sizes 128, 256 and 512, one query token to whole packed prompts, every mask, cells that must stay as
they were, pages shared by sequences, strided operands, a captured graph, another stream, and a run of the operators
together: decode, weights, eviction, decode over what stayed.

Bound of a weight 2^(t - lse), with lse an input: the score t is a sum of hs products whose query factor is held to
2^-22 and which is added up in fp32 (2^-24 of the sum of magnitudes a step, a step per 16 products; 2^-20 of that sum
covers both), and the exponential's argument and value are rounded to fp32; relative to the weight that is
ln 2 x 2^-20 x sum |q k| c, plus 2^-23 x |lse| and 1e-5 for the exponential and the fp32 sums."""
import numpy as np
import pytest
import torch

from oracle import quantpack_oracle as qo
from vllm_quantpack_b200 import _lib
from vllm_quantpack_b200.attention import ops

import qp_testutil as U

pytestmark = pytest.mark.gpu
LOG2E = 1.4426950408889634


@pytest.fixture(autouse=True)
def no_device_error():
    yield
    assert _lib.device_error() == 0


def setup(device, fmt, hs, lens, nkv=2, seed=0, bs=16, **fill):
    table, nblocks = U.block_tables(lens, bs, seed=seed + 1)
    cache = U.Cache(fmt, nblocks, bs, device, nkv=nkv, hs=hs)
    for i, n in enumerate(lens):
        if n:
            cache.fill(table[i], n, seed=seed + 10 + i, **fill)
    return cache, table


def scores(cache, data, row_table, q_bits, n, dtype="bf16", after=0, window=0, softcap=0.0):
    """(tokens, heads, n) base-2 scores with -inf where masked, and the largest sum |q k| c, in fp64."""
    hs, nkv = cache.hs, cache.nkv
    K, _ = qo.read_sequence(data, cache.layout, row_table, n)           # (n, KV heads, hs)
    q = qo.single_rht(qo.to_f32(q_bits, dtype), U.signs(hs)).astype(np.float64)
    ql, nq = q.shape[:2]
    c = hs ** -0.5 / hs * LOG2E
    kk = np.repeat(np.asarray(K, np.float64), nq // nkv, axis=1)
    t = np.einsum("qhc,khc->qhk", q, kk) * c
    mag = (np.einsum("qhc,khc->qhk", np.abs(q), np.abs(kk)) * c).max(initial=0.0)
    if softcap:
        t = softcap * LOG2E * np.tanh(t / (softcap * LOG2E))
    vis = n - ql + after + np.arange(ql)[:, None, None]
    pos = np.arange(n)[None, None]
    hidden = pos > vis
    if window:
        hidden |= pos <= vis - window
    return np.where(hidden, -np.inf, t), mag


def lse_of(t):
    m = t.max(-1, initial=-np.inf)
    safe = np.where(np.isfinite(m), m, 0.0)
    with np.errstate(divide="ignore"):
        return np.log2(np.exp2(t - safe[..., None]).sum(-1)) + safe


def run(device, cache, table, q_bits, qlens, lens, weights, lse, dtype="bf16", q=None, **kw):
    kc, vc, ks, vs = cache.views
    q = U.to_torch(q_bits, device, dtype) if q is None else q
    cu = torch.tensor(np.concatenate([[0], np.cumsum(qlens)]), dtype=torch.int32, device=device)
    ops.accumulate_attention_weights(
        q, kc, vc, weights, lse=lse, cu_seqlens_q=cu, max_seqlen_q=max(qlens),
        seqused_k=torch.tensor(lens, dtype=torch.int32, device=device), max_seqlen_k=max(lens),
        softmax_scale=cache.hs ** -0.5, block_table=torch.from_numpy(table).to(device), k_scale_cache=ks,
        v_scale_cache=vs, **kw)
    torch.cuda.synchronize()
    return weights


def start_weights(cache, device, seed=3):
    """Earlier weights, another value in every cell of the pool."""
    rng = np.random.default_rng(seed)
    w = rng.gamma(0.3, 1.0, (cache.nblocks, cache.nkv, cache.block_size)).astype(np.float32) + np.float32(1e-3)
    return torch.from_numpy(w).to(device).transpose(1, 2)


def expect(cache, table, q_bits, qlens, lens, before, dtype="bf16", sinks=None, drop=(), after=0, **feat):
    """The weights after the call (blocks, block size, KV heads) in fp64, the fp32 lse it takes, and the bound."""
    data, want = cache.host_bytes(), before.cpu().numpy().astype(np.float64)
    rtol, lses, at, added = 1e-5, [], 0, np.zeros_like(want)
    group = q_bits.shape[1] // cache.nkv
    for b, (ql, n) in enumerate(zip(qlens, lens)):
        qb = q_bits[at:at + ql]
        if ql == 0:
            continue
        if n == 0:
            lses.append(np.full((ql, q_bits.shape[1]), -np.inf, np.float32))
            at += ql
            continue
        t, mag = scores(cache, data, table[b], qb, n, dtype, after=after, **feat)
        lse = lse_of(t)
        if sinks is not None:
            lse = np.logaddexp2(lse, sinks[None] * LOG2E)
        lse = lse.astype(np.float32)
        for tok, head in drop:
            lse[tok, head] = -np.inf
        lses.append(lse)
        finite = np.where(np.isfinite(lse), lse, np.inf).astype(np.float64)
        w = np.exp2(t - finite[..., None]).reshape(ql, cache.nkv, group, n).sum((0, 2))   # (KV heads, n)
        pos = np.arange(n)
        blk, slot = np.asarray(table[b])[pos // cache.block_size], pos % cache.block_size
        own = pos >= n - ql + after
        want[blk[own], slot[own]] = 0.0
        np.add.at(want, (blk, slot), w.T)
        np.add.at(added, (blk, slot), w.T)
        big = np.abs(lse[np.isfinite(lse)]).max(initial=0.0)
        rtol = max(rtol, 1e-5 + np.log(2) * 2.0 ** -20 * mag + 2.0 ** -23 * big)
        at += ql
    return want, np.concatenate(lses), rtol, added


def check(device, fmt, hs, nq, nkv, qlens, lens, dtype="bf16", seed=0, kw=None, bs=16, fill=None, sinks=None, drop=()):
    kw = kw or {}
    cache, table = setup(device, fmt, hs, lens, nkv=nkv, seed=seed, bs=bs, **(fill or {}))
    qb = U.make_queries(qlens, seed=seed + 5, nq=nq, hs=hs, dtype=dtype)
    before = start_weights(cache, device)
    feat = {"window": kw.get("sliding_window", 0), "softcap": kw.get("softcap", 0.0),
            "after": kw.get("tokens_after_keys", 0)}
    want, lse, rtol, added = expect(cache, table, qb, qlens, lens, before, dtype, sinks=sinks, drop=drop, **feat)
    got = run(device, cache, table, qb, qlens, lens, before.clone(), torch.from_numpy(lse).to(device), dtype, **kw)
    got = got.cpu().numpy()
    same = added == 0.0
    err = np.abs(got - want)
    # fp32 storage rounds old + new once (2^-24); a weight below fp32's normal range is lost whole
    assert (err <= rtol * added + 2.0 ** -23 * np.abs(want) + 1e-37).all(), (err / (np.abs(want) + 1e-30)).max()
    own_zero = want == 0.0
    untouched = same & ~own_zero
    assert np.array_equal(got[untouched], before.cpu().numpy()[untouched])


@pytest.mark.parametrize("fmt", ["int4", "k8v4"])
@pytest.mark.parametrize("hs,nq,nkv", [(128, 32, 8), (256, 24, 4), (512, 16, 2), (128, 3, 3), (256, 8, 1)])
@pytest.mark.parametrize("qlen", [1, 4])
def test_decode_steps(device, fmt, hs, nq, nkv, qlen):
    check(device, fmt, hs, nq, nkv, [qlen], [777], seed=1)


@pytest.mark.parametrize("fmt,hs", [("int4", 128), ("k8v4", 256)])
@pytest.mark.parametrize("n", [1, 2, 16, 127, 128, 129, 255, 256, 257, 5000])
def test_context_lengths(device, fmt, hs, n):
    check(device, fmt, hs, 8, 2, [1], [n], seed=2)


@pytest.mark.parametrize("fmt,hs,bs", [("int4", 256, 16), ("k8v4", 128, 48), ("int4", 128, 272)])
def test_ragged_batches(device, fmt, hs, bs):
    """Lengths that differ by orders, requests without queries or keys, pages that end inside a tile."""
    check(device, fmt, hs, 8, 2, [2, 1, 0, 4, 3, 1], [3001, 1, 40, 17, 900, 0], seed=3, bs=bs)


@pytest.mark.parametrize("fmt,hs,nq,nkv", [("int4", 128, 8, 2), ("k8v4", 128, 32, 8), ("int4", 256, 12, 2),
                                           ("k8v4", 256, 4, 4), ("int4", 512, 8, 2), ("k8v4", 512, 16, 2)])
def test_whole_prompts(device, fmt, hs, nq, nkv):
    """Packed prompts that score themselves: causal tiles of every shape."""
    lens = [300, 7, 513, 1]
    check(device, fmt, hs, nq, nkv, lens, lens, seed=4)


@pytest.mark.parametrize("fmt,hs", [("int4", 256), ("k8v4", 128), ("int4", 512)])
@pytest.mark.parametrize("qlen", [9, 33, 200])
def test_last_chunk_of_a_prompt(device, fmt, hs, qlen):
    check(device, fmt, hs, 12, 2, [qlen, 5], [1700, 260], seed=5)


@pytest.mark.parametrize("hs", [128, 256, 512])
@pytest.mark.parametrize("window,softcap,after", [(1, 0.0, 0), (50, 0.0, 0), (900, 30.0, 0), (0, 2.0, 0), (0, 0.0, 3),
                                                  (300, 0.0, 100), (20, 0.0, 5000)])
def test_masks_and_softcap(device, hs, window, softcap, after):
    kw = dict(sliding_window=window, softcap=softcap, tokens_after_keys=after)
    check(device, "int4", hs, 8, 2, [4, 1], [1000, 300], seed=6, kw=kw)
    check(device, "k8v4", hs, 8, 2, [150, 40], [600, 40], seed=7, kw=kw)


def test_sinks_rows_without_lse_fp16_and_spreading_keys(device):
    nq = 8
    check(device, "int4", 256, nq, 2, [4], [500], dtype="fp16", seed=8, sinks=np.linspace(-3, 6, nq),
          drop=[(0, 1), (2, 7)])
    check(device, "k8v4", 128, nq, 2, [40], [500], dtype="fp16", seed=9, drop=[(0, 0), (39, 7), (5, 3)])
    check(device, "int4", 128, nq, 2, [2], [900], seed=10, fill=dict(spread=1.0))


def test_strided_operands(device):
    """Queries as a slice of a wider projection, rotated beforehand; weights with the KV heads innermost."""
    hs, nq, nkv, lens, qlens = 128, 8, 2, [700, 60], [2, 1]
    cache, table = setup(device, "int4", hs, lens, nkv=nkv, seed=11)
    qb = U.make_queries(qlens, seed=12, nq=nq, hs=hs)
    before = start_weights(cache, device).contiguous()
    want, lse, rtol, added = expect(cache, table, qb, qlens, lens, before)
    wide = torch.zeros((3, nq + 4, hs), dtype=torch.bfloat16, device=device)
    wide[:, :nq] = U.to_torch(qb, device)
    got = run(device, cache, table, qb, qlens, lens, before.clone(), torch.from_numpy(lse).to(device), q=wide[:, :nq])
    err = np.abs(got.cpu().numpy() - want)
    assert (err <= rtol * added + 2.0 ** -23 * np.abs(want)).all()


def test_shared_pages_get_every_sequence(device):
    """Two requests over one prompt's pages: a cell's weight is the sum of both."""
    hs, nq, nkv, n = 256, 8, 2, 320
    cache, table = setup(device, "int4", hs, [n], nkv=nkv, seed=13)
    table2 = np.repeat(table, 2, axis=0)
    qb = U.make_queries([1, 1], seed=14, nq=nq, hs=hs)
    before = torch.zeros((cache.nblocks, nkv, 16), device=device).transpose(1, 2)
    both = np.zeros((cache.nblocks, 16, nkv))
    lses = []
    for b in range(2):
        want, lse, rtol, added = expect(cache, table, qb[b:b + 1], [1], [n], before, after=1)
        both += want
        lses.append(lse)
    got = run(device, cache, table2, qb, [1, 1], [n, n], before.clone(),
              torch.from_numpy(np.concatenate(lses)).to(device), tokens_after_keys=1)
    assert np.allclose(got.cpu().numpy(), both, rtol=2 * rtol, atol=1e-30)


def test_captured_graph_and_other_stream(device):
    hs, nq, nkv, lens, qlens = 256, 24, 4, [1500, 90], [4, 2]
    cache, table = setup(device, "int4", hs, lens, nkv=nkv, seed=15)
    qb = U.make_queries(qlens, seed=16, nq=nq, hs=hs)
    before = start_weights(cache, device)
    want, lse, rtol, added = expect(cache, table, qb, qlens, lens, before)
    q, lse_t = U.to_torch(qb, device), torch.from_numpy(lse).to(device)
    kc, vc, ks, vs = cache.views
    args = dict(cu_seqlens_q=torch.tensor([0, 4, 6], dtype=torch.int32, device=device), max_seqlen_q=4,
                seqused_k=torch.tensor(lens, dtype=torch.int32, device=device), max_seqlen_k=max(lens),
                softmax_scale=hs ** -0.5, block_table=torch.from_numpy(table).to(device), k_scale_cache=ks,
                v_scale_cache=vs)
    weights = before.clone()
    ops.accumulate_attention_weights(q, kc, vc, before.clone(), lse=lse_t, **args)   # sizes the workspace
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.accumulate_attention_weights(q, kc, vc, weights, lse=lse_t, **args)
    weights.copy_(before)
    graph.replay()
    torch.cuda.synchronize()
    assert (np.abs(weights.cpu().numpy() - want) <= rtol * added + 2.0 ** -23 * np.abs(want)).all()
    side, again = torch.cuda.Stream(), before.clone()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.accumulate_attention_weights(q, kc, vc, again, lse=lse_t, **args)
    side.synchronize()
    assert torch.equal(again, weights)


@pytest.mark.parametrize("fmt,hs,nq,nkv", [("int4", 128, 8, 2), ("k8v4", 256, 12, 2), ("int4", 512, 8, 2)])
def test_score_evict_attend(device, fmt, hs, nq, nkv):
    """The operators together: decode with its log-sum-exp, weights of every key, eviction in place, and the next
    decode, which must equal attention over exactly the kept keys of each KV head."""
    lens, qlens, keep, first, last = [900, 333, 60], [1, 1, 1], 256, 4, 100
    cache, table = setup(device, fmt, hs, lens, nkv=nkv, seed=17)
    data = cache.host_bytes()
    qb = U.make_queries(qlens, seed=18, nq=nq, hs=hs)
    kc, vc, ks, vs = cache.views
    q = U.to_torch(qb, device)
    used = torch.tensor(lens, dtype=torch.int32, device=device)
    bt = torch.from_numpy(table).to(device)
    args = dict(cu_seqlens_q=torch.arange(4, dtype=torch.int32, device=device), max_seqlen_q=1,
                softmax_scale=hs ** -0.5, block_table=bt, k_scale_cache=ks, v_scale_cache=vs)
    lse = torch.empty((3, nq), dtype=torch.float32, device=device)
    ops.paged_decode(q, kc, vc, torch.empty_like(q), seqused_k=used, max_seqlen_k=900, lse_out=lse, **args)
    weights = ops.new_attention_weights(ks)
    ops.accumulate_attention_weights(q, kc, vc, weights, lse=lse, seqused_k=used, max_seqlen_k=900, **args)
    total = weights.sum().item()
    # every row hands out a weight of 1, to the attention's own accuracy (its scores: 2^-12 of a few units)
    assert abs(total - 3 * nq) < 0.01 * 3 * nq
    before = weights.clone()
    kept, new = ops.evict_cache(kc, vc, weights, seqused_k=used, max_seqlen_k=900, block_table=bt, keep=keep,
                                keep_first=first, keep_last=last, k_scale_cache=ks, v_scale_cache=vs)
    assert new.tolist() == [256, 256, 60]
    out = torch.empty_like(q)
    ops.paged_decode(q, kc, vc, out, seqused_k=new, max_seqlen_k=256, **args)
    torch.cuda.synchronize()
    group, sg = nq // nkv, U.signs(hs)
    q_rot = qo.single_rht(qo.to_f32(qb, "bf16"), sg).astype(np.float64)
    want = np.zeros((3, nq, hs))
    for b, n in enumerate(lens):
        K, V = qo.read_sequence(data, cache.layout, table[b], n)
        for h in range(nkv):
            idx = kept[b, h].cpu().numpy()
            idx = idx[idx >= 0]
            if n > keep:    # the choice itself
                w = before[bt[b].long()].flatten(0, 1)[:n, h].cpu().numpy()
                mid = np.arange(first, n - last)
                best = mid[np.argsort(-w[mid], kind="stable")[:keep - first - last]]
                assert np.array_equal(idx, np.sort(np.concatenate([np.arange(first), best, np.arange(n - last, n)])))
            else:
                assert np.array_equal(idx, np.arange(n))
            rows = q_rot[b, h * group:(h + 1) * group]
            t = rows @ np.asarray(K, np.float64)[idx, h].T * hs ** -1.5
            p = np.exp(t - t.max(-1, keepdims=True))
            o = p @ np.asarray(V, np.float64)[idx, h] / p.sum(-1, keepdims=True)
            want[b, h * group:(h + 1) * group] = qo.single_rht(o.astype(np.float32), sg, inverse=True) / hs
    assert qo.relerr(out.float().cpu().numpy(), want) < 5e-3


@pytest.mark.parametrize("fmt,qlens,lens", [("k8v4", [150], [700]), ("int4", [3] * 40, list(range(3, 363, 9)))])
def test_query_records_change_hands(device, fmt, qlens, lens):
    """Head 512, where the ring holds one query record: it is copied over as soon as the summing warps have given the
    one before back, in the middle of masked tiles (a window, causal ends). A key's sum has a fixed order, so twenty
    calls give the same bits, within the bound of the definition."""
    cache, table = setup(device, fmt, 512, lens, nkv=1, seed=31)
    qb = U.make_queries(qlens, seed=32, nq=8, hs=512)
    before = start_weights(cache, device)
    want, lse, rtol, added = expect(cache, table, qb, qlens, lens, before, window=100)
    lse = torch.from_numpy(lse).to(device)
    first = None
    for _ in range(20):
        got = run(device, cache, table, qb, qlens, lens, before.clone(), lse, sliding_window=100)
        if first is None:
            first = got
            err = np.abs(got.cpu().numpy() - want)
            assert (err <= rtol * added + 2.0 ** -23 * np.abs(want) + 1e-37).all()
        assert torch.equal(got, first)


@pytest.mark.parametrize("fmt,hs", [("int4", 128), ("k8v4", 256)])
def test_long_prompt_of_alike_weights(device, fmt, hs):
    """A prompt of 16,384 tokens whose rows give every key they see the same weight (zero queries, one lse): up to
    131,072 equal additions a key, whose roundings all fall the same way where they are added one by one.

    Bound, relative, whatever the rows: the exponential 2^-22; a tile of 64 rows is added up in two chains of 32, 31 x
    2^-24 (half a step each); the sum over the tiles is compensated, 2 x 2^-24; the two chains 2^-24; the parts of a group
    that several CTAs share are added in 64 bits, 2^-24 for the result."""
    n, nq, lse_value = 16384, 8, np.float32(1.7)
    cache, table = setup(device, fmt, hs, [n], nkv=1, seed=41)
    q = torch.zeros((n, nq, hs), dtype=torch.bfloat16, device=device)
    lse = torch.full((n, nq), float(lse_value), device=device)
    got = run(device, cache, table, None, [n], [n], start_weights(cache, device), lse, q=q)
    got = got.cpu().numpy()[table[0]].reshape(-1)[:n]
    want = nq * (n - np.arange(n, dtype=np.float64)) * np.exp2(-np.float64(lse_value))
    rel = np.abs(got / want - 1)
    assert rel.max() <= 2.0 ** -22 + (31 + 2 + 1 + 1) * 2.0 ** -24, rel.max()


@pytest.mark.parametrize("fmt,hs", [("int4", 128), ("k8v4", 256), ("int4", 512)])
@pytest.mark.parametrize("qlen", [1, 30])
def test_nan_in_cells_no_row_sees(device, fmt, hs, qlen):
    """Cells in front of every row's window hold NaN scales (their pages may be another's by now): they get nothing,
    and the tile's other keys what is theirs."""
    n, window = 903, 77
    cache, table = setup(device, fmt, hs, [n], nkv=2, seed=43)
    qb = U.make_queries([qlen], seed=44, nq=6, hs=hs)
    before = start_weights(cache, device)
    want, lse, rtol, added = expect(cache, table, qb, [qlen], [n], before, window=window)
    raw = cache.phys.view(torch.uint8)
    for i in range(n - qlen + 1 - window):
        raw[int(table[0][i // 16]), :, i % 16] = 0xFF
    got = run(device, cache, table, qb, [qlen], [n], before.clone(), torch.from_numpy(lse).to(device),
              sliding_window=window).cpu().numpy()
    assert np.isfinite(got).all()
    assert (np.abs(got - want) <= rtol * added + 2.0 ** -23 * np.abs(want) + 1e-37).all()


@pytest.mark.parametrize("prompt", [1, 150])
def test_nine_hundred_requests(device, prompt):
    """More requests than a CTA has threads, with some that have no query or no key among them: the scans that find a
    CTA's share and a query tile's place go on from one round of threads to the next. Few rows, and with a prompt of
    several tiles near the end."""
    rng = np.random.default_rng(45)
    lens = [int(n) for n in rng.integers(0, 50, 900)]
    qlens = [min(int(rng.integers(0, 3)), n) if n else int(rng.integers(0, 2)) for n in lens]
    lens[880], qlens[880] = 700, prompt
    check(device, "int4", 128, 8, 2, qlens, lens, seed=46)
