"""Head 128 (the size of most models' attention) on the split-KV kernel's register path (csrc/qp_decode128.cu), both
cache formats, against the fp64 oracle computed from the same cache bytes: every count of 8-row query blocks, single
tokens to long contexts, ends inside a 16-cell run and a page, ragged batches, split counts, page sizes, fp16,
strided queries, spreading and rising magnitudes (the rescale paths), rows that see no key, pages that hold NaN
scales behind the sequence, sliding windows, softcap, sinks, the varlen launch, chunk prefill, a sequence split, the
static-scratch decode, a captured graph, another stream, and the log-sum-exp output.

Bound: a row's error relative to its norm is at most about 2^-8 (the bf16 output) + 2^-11 (P in fp16) + the scores'
error (q in fp16: 2^-12 of a few units) in the worst case, and under half of that in the 2-norm: 5e-3, as at the
other head sizes. A log-sum-exp moves by at most the largest error of a score: 2^-12 x sum |q k| scale log2 e, about
10 units for these inputs times the outlier channels' 3: 0.01."""
import numpy as np
import pytest
import torch

from oracle import quantpack_oracle as qo
from vllm_quantpack_b200 import _lib
from vllm_quantpack_b200.attention import ops, rht
from vllm_quantpack_b200.attention import seq_parallel as sp

import qp_testutil as U

pytestmark = pytest.mark.gpu
HS = 128
TOL, LSE_TOL = 5e-3, 0.01


@pytest.fixture(autouse=True)
def no_device_error():
    yield
    assert _lib.device_error() == 0


def setup(device, fmt, lens, seed=0, bs=16, nkv=4, **fill):
    table, nblocks = U.block_tables(lens, bs, seed=seed + 1)
    cache = U.Cache(fmt, nblocks, bs, device, nkv=nkv, hs=HS)
    for i, n in enumerate(lens):
        cache.fill(table[i], n, seed=seed + 10 + i, **fill)
    return cache, table


def check(cache, table, q_bits, qlens, lens, got, dtype="bf16", **kw):
    want = U.reference(cache.host_bytes(), cache.layout, q_bits, qlens, lens, table, dtype=dtype, **kw)
    err = qo.relerr(got, want)
    assert err < TOL, f"relative error {err:.3e}"


@pytest.mark.parametrize("fmt", ["int4", "k8v4"])
@pytest.mark.parametrize("group,qlen", [(1, 1), (4, 1), (8, 1), (4, 3), (5, 3), (6, 4), (8, 4), (32, 1)],
                         ids=lambda v: str(v))
def test_rows_per_kv_head(device, fmt, group, qlen):
    """1 to 32 query rows: each of the kernel's four row-block counts, full and ragged."""
    lens, nkv = [777], 2
    cache, table = setup(device, fmt, lens, nkv=nkv)
    qb = U.make_queries([qlen], seed=3, nq=group * nkv, hs=HS)
    check(cache, table, qb, [qlen], lens, U.decode(cache, qb, [qlen], lens, table))


@pytest.mark.parametrize("fmt", ["int4", "k8v4"])
@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 31, 32, 33, 255, 256, 257, 1000, 8191])
def test_context_lengths(device, fmt, n):
    cache, table = setup(device, fmt, [n], seed=1)
    qb = U.make_queries([1], seed=4, nq=16, hs=HS)
    check(cache, table, qb, [1], [n], U.decode(cache, qb, [1], [n], table))


@pytest.mark.parametrize("fmt,bs,splits", [("int4", 16, 1), ("int4", 48, 3), ("k8v4", 32, 7), ("k8v4", 528, 33),
                                           ("int4", 16, 200)])
def test_splits_and_page_sizes(device, fmt, bs, splits):
    """One split over everything, odd splits, more splits than 32-key tiles; pages that end inside a tile."""
    lens, qlens = [3001, 40, 1200], [2, 4, 1]
    cache, table = setup(device, fmt, lens, seed=2, bs=bs)
    qb = U.make_queries(qlens, seed=5, nq=16, hs=HS)
    check(cache, table, qb, qlens, lens, U.decode(cache, qb, qlens, lens, table, num_splits=splits))


@pytest.mark.parametrize("fmt", ["int4", "k8v4"])
def test_ragged_batch_and_long_context(device, fmt):
    lens, qlens = [70000, 1, 513, 9000, 64], [4, 1, 3, 2, 4]
    cache, table = setup(device, fmt, lens, seed=3)
    qb = U.make_queries(qlens, seed=6, nq=24, hs=HS)
    check(cache, table, qb, qlens, lens, U.decode(cache, qb, qlens, lens, table))


@pytest.mark.parametrize("fmt", ["int4", "k8v4"])
@pytest.mark.parametrize("spread,grow", [(2.0, 0.0), (0.0, 30.0), (1.0, 10.0)])
def test_spreading_and_rising_magnitudes(device, fmt, spread, grow):
    """Keys and values whose magnitudes differ by orders inside a tile and rise along the context: the running
    maximum and the rows' value factors change many times."""
    lens, qlens = [4000], [4]
    cache, table = setup(device, fmt, lens, seed=4, spread=spread, grow=grow)
    qb = U.make_queries(qlens, seed=7, nq=16, hs=HS)
    for splits in (1, 9):
        check(cache, table, qb, qlens, lens, U.decode(cache, qb, qlens, lens, table, num_splits=splits))


@pytest.mark.parametrize("fmt", ["int4", "k8v4"])
def test_fp16_strided_queries_and_lse(device, fmt):
    """fp16, queries and output as slices of wider rows (a fused projection), and the log-sum-exp beside them."""
    lens, qlens, nq, nkv = [3000, 411], [2, 1], 8, 2
    cache, table = setup(device, fmt, lens, seed=5, nkv=nkv)
    qb = U.make_queries(qlens, seed=8, nq=nq, hs=HS, dtype="fp16")
    wide = torch.zeros((3, nq + 2 * nkv, HS), dtype=torch.float16, device=device)
    wide[:, :nq] = U.to_torch(qb, device, "fp16")
    holder = torch.full((3, nq + 1, HS), 7.0, dtype=torch.float16, device=device)
    kc, vc, ks, vs = cache.views
    lse = torch.empty((3, nq), dtype=torch.float32, device=device)
    ops.paged_decode(wide[:, :nq], kc, vc, holder[:, :nq],
                     cu_seqlens_q=torch.tensor([0, 2, 3], dtype=torch.int32, device=device), max_seqlen_q=2,
                     seqused_k=torch.tensor(lens, dtype=torch.int32, device=device), max_seqlen_k=max(lens),
                     softmax_scale=HS ** -0.5, block_table=torch.from_numpy(table).to(device), k_scale_cache=ks,
                     v_scale_cache=vs, lse_out=lse)
    check(cache, table, qb, qlens, lens, holder[:, :nq].float().cpu().numpy(), dtype="fp16")
    assert (holder[:, nq:] == 7.0).all()
    want = oracle_lse(cache, table, qb, qlens, lens, "fp16")
    assert np.abs(lse.cpu().numpy() - want).max() < LSE_TOL


def oracle_lse(cache, table, q_bits, qlens, lens, dtype="bf16"):
    """Base-2 log-sum-exp of every row (tokens, query heads)."""
    data, sg, out, at = cache.host_bytes(), U.signs(cache.hs), [], 0
    for i, (ql, n) in enumerate(zip(qlens, lens)):
        q_rot = qo.single_rht(qo.to_f32(q_bits[at:at + ql], dtype), sg).astype(np.float64)
        out.append(qo.attention_from_cache(q_rot, data, cache.layout, table[i], n, cache.hs ** -0.5)[1])
        at += ql
    return np.concatenate(out) / np.log(2.0)


@pytest.mark.parametrize("hs,nq,nkv", [(256, 24, 4), (512, 16, 2)])
def test_lse_output_at_the_other_head_sizes(device, hs, nq, nkv):
    lens, qlens = [2000, 77], [4, 1]
    table, nblocks = U.block_tables(lens, 16, seed=9)
    cache = U.Cache("int4", nblocks, 16, device, nkv=nkv, hs=hs)
    for i, n in enumerate(lens):
        cache.fill(table[i], n, seed=20 + i)
    qb = U.make_queries(qlens, seed=9, nq=nq, hs=hs)
    q = U.to_torch(qb, device)
    kc, vc, ks, vs = cache.views
    common = dict(cu_seqlens_q=torch.tensor([0, 4, 5], dtype=torch.int32, device=device),
                  seqused_k=torch.tensor(lens, dtype=torch.int32, device=device), max_seqlen_k=max(lens),
                  softmax_scale=hs ** -0.5, block_table=torch.from_numpy(table).to(device), k_scale_cache=ks,
                  v_scale_cache=vs)
    want = oracle_lse(cache, table, qb, qlens, lens)
    out, plain = torch.empty_like(q), torch.empty_like(q)
    ops.paged_decode(q, kc, vc, plain, max_seqlen_q=4, **common)
    for fn, kw in ((ops.paged_decode, dict(max_seqlen_q=4)), (ops.prefill_varlen, {})):
        lse = torch.empty((5, nq), dtype=torch.float32, device=device)
        fn(q, kc, vc, out, lse_out=lse, **kw, **common)
        assert np.abs(lse.cpu().numpy() - want).max() < LSE_TOL
        if fn is ops.paged_decode:
            assert torch.equal(out, plain)   # the output is the one without it
    # a chunk prefill's rows
    chunk = U.make_queries([70], seed=10, nq=nq, hs=hs)
    lse = torch.empty((70, nq), dtype=torch.float32, device=device)
    qc = U.to_torch(chunk, device)
    ops.prefill(qc, kc, vc, torch.empty_like(qc), block_row=torch.from_numpy(table[0]).to(device), n=lens[0],
                softmax_scale=hs ** -0.5, k_scale_cache=ks, v_scale_cache=vs, lse_out=lse)
    want = oracle_lse(cache, table, chunk, [70], lens[:1])
    assert np.abs(lse.cpu().numpy() - want).max() < LSE_TOL


@pytest.mark.parametrize("fmt", ["int4", "k8v4"])
@pytest.mark.parametrize("window,softcap,sink", [(1, 0.0, False), (40, 0.0, False), (700, 50.0, False),
                                                 (0, 3.0, True), (5000, 0.0, True), (33, 3.0, True)])
def test_layer_features(device, fmt, window, softcap, sink):
    lens, qlens, nq = [2100, 17, 900], [4, 2, 1], 16
    cache, table = setup(device, fmt, lens, seed=6)
    qb = U.make_queries(qlens, seed=11, nq=nq, hs=HS)
    sinks = np.linspace(-4, 9, nq).astype(np.float32) if sink else None
    kw = dict(sliding_window=window, softcap=softcap, sinks=sinks)
    for splits in (None, 5):
        check(cache, table, qb, qlens, lens, U.decode(cache, qb, qlens, lens, table, num_splits=splits, **kw), **kw)


@pytest.mark.parametrize("fmt", ["int4", "k8v4"])
def test_rows_without_keys_and_garbage_behind(device, fmt):
    """A sequence shorter than its query tokens: the rows before its first key give 0 and an lse of -inf. The pages'
    unwritten cells hold NaN scales and must reach nothing."""
    lens, qlens, nq = [2, 50, 0], [4, 1, 1], 8
    table, nblocks = U.block_tables([16, 64, 16], 16, seed=7)
    cache = U.Cache(fmt, nblocks, 16, device, nkv=2, hs=HS)
    cache.phys.view(torch.uint8).fill_(0xFF)    # scale words of NaN, codes of all ones
    for i, n in enumerate(lens):
        if n:
            cache.fill(table[i], n, seed=30 + i)
    qb = U.make_queries(qlens, seed=12, nq=nq, hs=HS)
    kc, vc, ks, vs = cache.views
    q = U.to_torch(qb, device)
    out = torch.full_like(q, float("nan"))
    lse = torch.full((6, nq), float("nan"), dtype=torch.float32, device=device)
    ops.paged_decode(q, kc, vc, out, cu_seqlens_q=torch.tensor([0, 4, 5, 6], dtype=torch.int32, device=device),
                     max_seqlen_q=4, seqused_k=torch.tensor(lens, dtype=torch.int32, device=device), max_seqlen_k=64,
                     softmax_scale=HS ** -0.5, block_table=torch.from_numpy(table).to(device), k_scale_cache=ks,
                     v_scale_cache=vs, lse_out=lse)
    got = out.float().cpu().numpy()
    assert (got[:2] == 0).all() and (got[5] == 0).all()
    assert torch.isinf(lse[:2]).all() and torch.isinf(lse[5]).all()
    data = cache.host_bytes()
    want = np.concatenate([U.reference(data, cache.layout, qb[2:4], [2], [2], table[:1]),
                           U.reference(data, cache.layout, qb[4:5], [1], [50], table[1:2])])
    assert qo.relerr(got[2:5], want) < TOL


@pytest.mark.parametrize("fmt", ["int4", "k8v4"])
def test_varlen_and_chunk_prefill(device, fmt):
    qlens, lens, nq = [100, 7, 33], [1500, 7, 33], 16
    cache, table = setup(device, fmt, lens, seed=8)
    qb = U.make_queries(qlens, seed=13, nq=nq, hs=HS)
    kc, vc, ks, vs = cache.views
    q = U.to_torch(qb, device)
    out = torch.empty_like(q)
    ops.prefill_varlen(q, kc, vc, out, cu_seqlens_q=torch.tensor([0, 100, 107, 140], dtype=torch.int32, device=device),
                       seqused_k=torch.tensor(lens, dtype=torch.int32, device=device), max_seqlen_k=max(lens),
                       block_table=torch.from_numpy(table).to(device), softmax_scale=HS ** -0.5, k_scale_cache=ks,
                       v_scale_cache=vs)
    check(cache, table, qb, qlens, lens, out.float().cpu().numpy())
    out = torch.empty_like(q[:100])
    ops.prefill(q[:100], kc, vc, out, block_row=torch.from_numpy(table[0]).to(device), n=lens[0],
                softmax_scale=HS ** -0.5, k_scale_cache=ks, v_scale_cache=vs)
    check(cache, table[:1], qb[:100], [100], lens[:1], out.float().cpu().numpy())


def test_sequence_split_folds_to_the_whole(device):
    """Two ranges of one sequence as two ranks hold them (tokens after the keys, a window that reaches into the
    earlier range): fp32 partials and their base-2 lse, folded."""
    n, qlen, nq, world = 3008, 4, 16, 2
    cache, table = setup(device, "int4", [n], seed=9)
    qb = U.make_queries([qlen], seed=14, nq=nq, hs=HS)
    kc, vc, ks, vs = cache.views
    q = U.to_torch(qb, device)
    for window in (0, 1700):
        part_o = torch.empty((world, qlen, nq, HS), dtype=torch.float32, device=device)
        part_lse = torch.empty((world, qlen, nq), dtype=torch.float32, device=device)
        for r in range(world):
            lo, hi, after = sp.sequence_range(n, r, world)
            ops.paged_decode(q, kc, vc, part_o[r], cu_seqlens_q=torch.tensor([0, qlen], dtype=torch.int32, device=device),
                             max_seqlen_q=qlen, seqused_k=torch.tensor([hi - lo], dtype=torch.int32, device=device),
                             max_seqlen_k=hi - lo, softmax_scale=HS ** -0.5, k_scale_cache=ks, v_scale_cache=vs,
                             block_table=torch.from_numpy(table[:, lo // 16:(hi + 15) // 16].copy()).to(device),
                             out_fp32_lse=part_lse[r], tokens_after_keys=after, sliding_window=window)
        out = torch.empty_like(q)
        ops.merge_attn_partials(part_o, part_lse, out)
        check(cache, table, qb, [qlen], [n], out.float().cpu().numpy(), sliding_window=window)


def test_static_scratch_graph_and_stream(device):
    """The decode without a workspace equals the one with it; a captured decode replays over new queries and lengths;
    a call on another stream gives the same rows."""
    lens, qlens, nq = [900, 33], [1, 1], 16
    cache, table = setup(device, "k8v4", lens, seed=10)
    qb = U.make_queries(qlens, seed=15, nq=nq, hs=HS)
    kc, vc, ks, vs = cache.views
    q = U.to_torch(qb, device)
    bt = torch.from_numpy(table).to(device)
    cu = torch.tensor([0, 1, 2], dtype=torch.int32, device=device)
    used = torch.tensor(lens, dtype=torch.int32, device=device)

    def decode(out):
        return ops.paged_decode(q, kc, vc, out, cu_seqlens_q=cu, max_seqlen_q=1, seqused_k=used, max_seqlen_k=900,
                                softmax_scale=HS ** -0.5, block_table=bt, k_scale_cache=ks, v_scale_cache=vs)

    want = decode(torch.empty_like(q))
    lay = ops.CacheLayout.of(kc, vc, ks, vs, HS)
    out = torch.empty_like(q)
    splits = ops.decode_num_splits(2, 4, 900, ops.sm_count(device))
    _lib.call("qp_paged_decode_static", lay.fmt, 0, q.data_ptr(), q.stride(0), q.stride(1), out.data_ptr(),
              out.stride(0), out.stride(1), 2, 2, cu.data_ptr(), used.data_ptr(), 1, bt.data_ptr(), bt.stride(0),
              *lay.args(), nq, 4, HS, HS ** -0.5, rht.device_sign_bits(HS, device).data_ptr(), 0, 0, None, splits,
              torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert qo.relerr(out.float().cpu().numpy(), want.float().cpu().numpy()) < TOL
    graph, captured = torch.cuda.CUDAGraph(), torch.empty_like(q)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        decode(captured)
    q2 = U.make_queries(qlens, seed=16, nq=nq, hs=HS)
    q.copy_(U.to_torch(q2, device))
    used.copy_(torch.tensor([850, 20], dtype=torch.int32))
    graph.replay()
    check(cache, table, q2, qlens, [850, 20], captured.float().cpu().numpy())
    side, other = torch.cuda.Stream(), torch.empty_like(q)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        decode(other)
    side.synchronize()
    assert torch.equal(other, captured)


@pytest.mark.parametrize("varlen", [False, True])
def test_rows_behind_the_last_sequence_stay(device, varlen):
    """A batch padded to a captured size: rows no sequence owns keep what they held, the output's and the lse's."""
    lens, qlens, nq, pad = [300, 40], [2, 1], 16, 5
    cache, table = setup(device, "int4", lens, seed=11)
    qb = U.make_queries([3 + pad], seed=17, nq=nq, hs=HS)
    q = U.to_torch(qb, device)
    kc, vc, ks, vs = cache.views
    out = torch.full_like(q, 3.0)
    lse = torch.full((3 + pad, nq), 5.0, dtype=torch.float32, device=device)
    args = dict(cu_seqlens_q=torch.tensor([0, 2, 3], dtype=torch.int32, device=device),
                seqused_k=torch.tensor(lens, dtype=torch.int32, device=device), max_seqlen_k=300,
                softmax_scale=HS ** -0.5, block_table=torch.from_numpy(table).to(device), k_scale_cache=ks,
                v_scale_cache=vs, lse_out=lse)
    if varlen:
        ops.prefill_varlen(q, kc, vc, out, **args)
    else:
        ops.paged_decode(q, kc, vc, out, max_seqlen_q=2, **args)
    assert (out[3:] == 3.0).all() and (lse[3:] == 5.0).all()
    check(cache, table, qb[:3], qlens, lens, out[:3].float().cpu().numpy())


def test_many_short_sequences_and_every_row_finite(device):
    """More (sequence, KV head) pairs than CTAs, most of them shorter than a tile: shares that cross many pairs."""
    rng = np.random.default_rng(12)
    lens = [int(n) for n in rng.integers(1, 90, 150)] + [3000]
    qlens = [min(4, n) for n in lens]
    cache, table = setup(device, "k8v4", lens, seed=12)
    qb = U.make_queries(qlens, seed=18, nq=8, hs=HS)
    for splits in (None, 2, 40):
        got = U.decode(cache, qb, qlens, lens, table, num_splits=splits)
        assert np.isfinite(got).all()
        check(cache, table, qb, qlens, lens, got)


def spoil(cache, table_row, positions):
    """NaN scales and codes of all ones in the cells of these positions."""
    raw = cache.phys.view(torch.uint8)
    for i in positions:
        raw[int(table_row[i // cache.block_size]), :, i % cache.block_size] = 0xFF


@pytest.mark.parametrize("fmt", ["int4", "k8v4"])
@pytest.mark.parametrize("splits", [None, 1])
def test_nan_in_cells_a_row_does_not_see(device, fmt, splits):
    """Cells in front of a sliding window (their pages may be another's by now) and the newest token's cell, which the
    earlier query tokens do not see, hold NaN: they reach no row that does not see them."""
    n, window, nq = 2101, 40, 16
    for qlen in (1, 3):
        cache, table = setup(device, fmt, [n], seed=52)
        qb = U.make_queries([qlen], seed=53, nq=nq, hs=HS)
        want = U.reference(cache.host_bytes(), cache.layout, qb, [qlen], [n], table, sliding_window=window)
        spoil(cache, table[0], range(n - qlen + 1 - window))
        got = U.decode(cache, qb, [qlen], [n], table, num_splits=splits, sliding_window=window)
        assert qo.relerr(got, want) < TOL
    cache, table = setup(device, fmt, [n], seed=54)
    qb = U.make_queries([4], seed=55, nq=nq, hs=HS)
    want = U.reference(cache.host_bytes(), cache.layout, qb, [4], [n], table)
    spoil(cache, table[0], [n - 1])
    got = U.decode(cache, qb, [4], [n], table, num_splits=splits)
    assert qo.relerr(got[:3], want[:3]) < TOL
    assert np.isnan(got[3]).all()


@pytest.mark.parametrize("fmt", ["int4", "k8v4"])
@pytest.mark.parametrize("drop", [20, 30])
@pytest.mark.parametrize("back", [False, True])
def test_values_shrink_while_scores_rise(device, fmt, drop, back):
    """The first keys hold values 2^drop times those of the later ones, whose scores pass them by about 80 (base 2): what
    the row is worth lies in the small values, which have to keep their digits (and, with `back`, in the large ones
    that come again at the end). The rows: one the scores rise for, one they fall for, one they rise half as far, a
    stranger."""
    n, lead, nq = 3000, 256, 4
    rng = np.random.default_rng(50)
    k0 = rng.standard_normal(HS).astype(np.float32)
    rise = np.where(np.arange(n) < lead, 0.01, rng.uniform(4.9, 5.0, n)).astype(np.float32)
    size = np.where(np.arange(n) < lead, 2.0 ** (drop - 20), 2.0 ** -20).astype(np.float32)
    if back:
        size[-40:] = size[0]
    kb = qo.from_f32(rise[:, None, None] * k0[None, None], "bf16")
    vb = qo.from_f32(size[:, None, None] * rng.standard_normal((n, 1, HS)).astype(np.float32), "bf16")
    table, nblocks = U.block_tables([n], 16, seed=51)
    cache = U.Cache(fmt, nblocks, 16, device, nkv=1, hs=HS)
    pos = np.arange(n)
    cache.store(kb, vb, table[0].astype(np.int64)[pos // 16] * 16 + pos % 16)
    qb = qo.from_f32(np.stack([k0, -k0, 0.5 * k0, rng.standard_normal(HS).astype(np.float32)])[None], "bf16")
    want = U.reference(cache.host_bytes(), cache.layout, qb, [1], [n], table)
    for splits in (1, 3):
        got = U.decode(cache, qb, [1], [n], table, num_splits=splits)
        for h in range(nq):     # each row by itself: their norms differ by 2^drop
            err = qo.relerr(got[:, h], want[:, h])
            assert err < TOL, f"row {h}, {splits} splits: relative error {err:.3e}"


@pytest.mark.parametrize("splits", [1, 5, 40])
def test_nan_query_row_and_its_lse(device, splits):
    """A row of NaN stays one, its log-sum-exp too (-inf says that a row sees no key); the other rows are untouched."""
    lens, qlens, nq = [3000], [2], 16
    cache, table = setup(device, "int4", lens, seed=56)
    qb = U.make_queries(qlens, seed=57, nq=nq, hs=HS)
    want, want_lse = U.reference(cache.host_bytes(), cache.layout, qb, qlens, lens, table), \
        oracle_lse(cache, table, qb, qlens, lens)
    kc, vc, ks, vs = cache.views
    q = U.to_torch(qb, device)
    q[1, 3] = float("nan")
    out, lse = torch.empty_like(q), torch.empty((2, nq), dtype=torch.float32, device=device)
    ops.paged_decode(q, kc, vc, out, cu_seqlens_q=torch.tensor([0, 2], dtype=torch.int32, device=device),
                     max_seqlen_q=2, seqused_k=torch.tensor(lens, dtype=torch.int32, device=device),
                     max_seqlen_k=lens[0], softmax_scale=HS ** -0.5, block_table=torch.from_numpy(table).to(device),
                     k_scale_cache=ks, v_scale_cache=vs, num_splits=splits, lse_out=lse)
    rest = np.ones((2, nq), bool)
    rest[1, 3] = False
    got, lse = out.float().cpu().numpy(), lse.cpu().numpy()
    assert np.isnan(got[1, 3]).all() and np.isnan(lse[1, 3])
    assert qo.relerr(got[rest], want[rest]) < TOL and np.abs(lse - want_lse)[rest].max() < LSE_TOL


def test_two_streams_at_once(device):
    """Decodes and weights of two requests on two streams, each with the default workspace: what one writes there is
    not the other's."""
    sides = [torch.cuda.Stream(), torch.cuda.Stream()]
    runs = []
    for i, n in enumerate((60000, 45000)):
        cache, table = setup(device, "int4", [n], seed=60 + i)
        q = U.to_torch(U.make_queries([2], seed=62 + i, nq=16, hs=HS), device)
        args = dict(cu_seqlens_q=torch.tensor([0, 2], dtype=torch.int32, device=device), max_seqlen_q=2,
                    seqused_k=torch.tensor([n], dtype=torch.int32, device=device), max_seqlen_k=n,
                    softmax_scale=HS ** -0.5, block_table=torch.from_numpy(table).to(device),
                    k_scale_cache=cache.views[2], v_scale_cache=cache.views[3])
        runs.append((cache, q, args))

    def step(i):
        cache, q, args = runs[i]
        out, lse = torch.empty_like(q), torch.empty((2, 16), dtype=torch.float32, device=device)
        weights = ops.new_attention_weights(cache.views[2])
        ops.paged_decode(q, *cache.views[:2], out, lse_out=lse, **args)
        ops.accumulate_attention_weights(q, *cache.views[:2], weights, lse=lse, **args)
        return out, lse, weights

    want = [step(i) for i in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(20):
        for i, side in enumerate(sides):
            with torch.cuda.stream(side):
                got.append((i, step(i)))
    torch.cuda.synchronize()
    for i, tensors in got:
        assert all(torch.equal(a, b) for a, b in zip(tensors, want[i]))


@pytest.mark.parametrize("tokens", [2, 4])
def test_nine_hundred_requests(device, tokens):
    """More requests than a CTA has threads, with some that have no query or no key among them and a long one near the
    end: the scan that finds a CTA's share goes on from one round of threads to the next."""
    rng = np.random.default_rng(58)
    lens = [int(n) for n in rng.integers(0, 60, 900)]
    qlens = [min(int(rng.integers(0, tokens + 1)), n) if n else int(rng.integers(0, 2)) for n in lens]
    lens[880], qlens[880], qlens[0], lens[0] = 5000, tokens, tokens, 40
    cache, table = setup(device, "int4", lens, seed=59, nkv=2)
    qb = U.make_queries(qlens, seed=60, nq=8, hs=HS)
    got = U.decode(cache, qb, qlens, lens, table)
    data, at = cache.host_bytes(), 0
    rows, want = [], []
    for i, (ql, n) in enumerate(zip(qlens, lens)):
        if ql and n:
            want.append(U.reference(data, cache.layout, qb[at:at + ql], [ql], [n], table[i:i + 1]))
            rows += range(at, at + ql)
        elif ql:
            assert (got[at:at + ql] == 0).all()
        at += ql
    want = np.concatenate(want)
    assert qo.relerr(got[rows], want) < TOL
    worst = np.linalg.norm(got[rows] - want, axis=-1) / np.linalg.norm(want, axis=-1)
    assert worst.max() < 4 * TOL    # no row is another's
