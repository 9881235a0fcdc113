"""Eviction by accumulated weight (csrc/qp_evict.cu) against a plain numpy form, byte for byte: the kept positions, the
new lengths, every byte of the pool and every weight, in place and into other pages."""
import numpy as np
import pytest
import torch

from vllm_quantpack_b200 import _lib
from vllm_quantpack_b200.attention import ops

import qp_testutil as U

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_device_error():
    yield
    assert _lib.device_error() == 0


def plain(pages, weights, table, lens, keep, first, last, out_table, block_size):
    """pages (blocks, block size, KV heads, cell) and weights (blocks, block size, KV heads), changed in place."""
    nkv = weights.shape[2]
    kept = np.full((len(lens), nkv, keep), -1, np.int32)
    old_pages, old_weights = pages.copy(), weights.copy()
    for b, n in enumerate(lens):
        pos = np.arange(n)
        src = table[b][pos // block_size], pos % block_size
        for h in range(nkv):
            w = old_weights[src[0], src[1], h]
            if n > keep:
                mid = np.arange(first, n - last)
                rank = np.where(np.isnan(w[mid]), -np.inf, w[mid] + 0.0)
                # NaN below everything, -inf included
                order = np.lexsort((mid, -rank, np.isnan(w[mid])))
                stay = np.sort(np.concatenate([np.arange(first), mid[order[:keep - first - last]],
                                               np.arange(n - last, n)])).astype(int)
            else:
                stay = pos
            kept[b, h, :len(stay)] = stay
            dst = table if out_table is None else out_table
            at = np.arange(len(stay))
            blk, slot = dst[b][at // block_size], at % block_size
            pages[blk, slot, h] = old_pages[src[0][stay], src[1][stay], h]
            weights[blk, slot, h] = w[stay]
    return kept, np.minimum(lens, keep)


def check(device, fmt, hs, nkv, lens, keep, first, last, out=False, bs=16, seed=0, make=None, nhd=False, alias=False,
          strided=False):
    rng = np.random.default_rng(seed)
    need = [(max(n, 1) + bs - 1) // bs for n in lens]
    width, wout = max(need), (keep + bs - 1) // bs
    total = len(lens) * (width + (wout if out else 0)) + 3
    order = rng.permutation(total).astype(np.int32)
    table = order[:len(lens) * width].reshape(len(lens), width)
    out_table = order[len(lens) * width:len(lens) * (width + wout)].reshape(len(lens), wout) if out else None
    cache = U.Cache(fmt, total, bs, device, nkv=nkv, hs=hs, nhd=nhd)
    raw = rng.integers(0, 256, cache.phys.shape, dtype=np.uint8)
    cache.phys.view(torch.uint8).copy_(torch.from_numpy(raw))
    w = (make(rng, (total, bs, nkv)) if make else rng.gamma(0.3, 1.0, (total, bs, nkv))).astype(np.float32)
    weights = torch.from_numpy(w).to(device)
    if not strided:
        weights = weights.transpose(1, 2).contiguous().transpose(1, 2)
    used = torch.tensor(lens, dtype=torch.int32, device=device)
    kc, vc, ks, vs = cache.views
    kept, new = ops.evict_cache(
        kc, vc, weights, seqused_k=used, max_seqlen_k=max(max(lens), 1), block_table=torch.from_numpy(table).to(device),
        keep=keep, keep_first=first, keep_last=last, k_scale_cache=ks, v_scale_cache=vs,
        out_block_table=None if out_table is None else torch.from_numpy(out_table).to(device),
        seqused_out=used if alias else None)
    torch.cuda.synchronize()
    pages = raw if nhd else raw.transpose(0, 2, 1, 3).copy()
    pages = pages.copy()
    want_kept, want_n = plain(pages, w, table, lens, keep, first, last, out_table, bs)
    assert np.array_equal(new.cpu().numpy(), want_n)
    assert np.array_equal(kept.cpu().numpy(), want_kept)
    got = cache.phys.view(torch.uint8).cpu().numpy()
    assert np.array_equal(got if nhd else got.transpose(0, 2, 1, 3), pages)
    assert np.array_equal(weights.cpu().numpy().view(np.uint32), w.view(np.uint32))
    if not alias:
        assert used.tolist() == list(lens)


@pytest.mark.parametrize("fmt,hs", [("int4", 128), ("k8v4", 128), ("int4", 256), ("k8v4", 256), ("int4", 512),
                                    ("k8v4", 512)])
@pytest.mark.parametrize("out", [False, True])
def test_formats(device, fmt, hs, out):
    check(device, fmt, hs, 3, [500, 77, 300], 200, 4, 50, out=out)


@pytest.mark.parametrize("out", [False, True])
@pytest.mark.parametrize("n,keep,first,last", [(2, 1, 0, 0), (2, 1, 1, 0), (2, 1, 0, 1), (17, 16, 4, 4), (300, 1, 0, 0),
                                               (300, 299, 0, 0), (300, 299, 200, 99), (1025, 1024, 4, 256),
                                               (4097, 64, 0, 64), (4097, 4000, 4000, 0), (3000, 1500, 0, 0),
                                               (3000, 2999, 1, 1)])
def test_sizes(device, n, keep, first, last, out):
    check(device, "int4", 128, 2, [n], keep, first, last, out=out, seed=n + keep)


@pytest.mark.parametrize("out", [False, True])
def test_batch_of_every_length(device, out):
    """Sequences below, at and above the budget, one token, none."""
    check(device, "k8v4", 128, 2, [1, 0, 99, 100, 101, 2000, 150, 5000], 100, 3, 20, out=out, seed=5)


@pytest.mark.parametrize("bs,nhd", [(16, True), (48, False), (272, True)])
def test_page_sizes_and_layouts(device, bs, nhd):
    check(device, "k8v4", 128, 3, [700, 90], 128, 2, 30, bs=bs, nhd=nhd, seed=6, strided=nhd)


def ties(rng, shape):
    return rng.integers(0, 3, shape)


def zeros(rng, shape):
    return np.where(rng.random(shape) < 0.5, -0.0, 0.0)


def odd(rng, shape):
    x = rng.normal(0, 1, shape)
    return np.choose(rng.integers(0, 6, shape), [x, np.inf, -np.inf, np.nan, 1e-42, -x])


@pytest.mark.parametrize("make", [ties, zeros, odd])
@pytest.mark.parametrize("n,keep", [(700, 300), (5000, 64), (5000, 4990)])
def test_equal_and_odd_weights(device, make, n, keep):
    """Ties go to the earlier token; infinities, NaN, denormals and both zeros keep their order."""
    check(device, "int4", 128, 2, [n, n - 7], keep, 5, 11, make=make, seed=n)
    check(device, "int4", 128, 2, [n, n - 7], keep, 0, 0, make=make, seed=n + 1, out=True)


def test_long_sequences(device):
    check(device, "int4", 128, 2, [70001, 300], 20000, 4, 1000, seed=8)
    check(device, "int4", 128, 1, [200003], 1000, 4, 100, out=True, seed=9)
    check(device, "int4", 128, 1, [450001], 300000, 4, 100, seed=10)


def test_lengths_in_place_graph_and_stream(device):
    check(device, "int4", 128, 2, [500, 40], 100, 0, 10, alias=True, seed=11)
    # captured: the second replay cuts what the first left (lengths read on the device each time)
    n, keep, nkv, hs = 600, 200, 2, 128
    table, nblocks = U.block_tables([n], 16, seed=2)
    cache = U.Cache("int4", nblocks, 16, device, nkv=nkv, hs=hs)
    rng = np.random.default_rng(3)
    raw = torch.from_numpy(rng.integers(0, 256, cache.phys.shape, dtype=np.uint8)).to(device)
    w0 = torch.from_numpy(rng.gamma(0.3, 1.0, (nblocks, nkv, 16)).astype(np.float32)).to(device)
    weights, used = w0.clone().transpose(1, 2), torch.tensor([n], dtype=torch.int32, device=device)
    bt = torch.from_numpy(table).to(device)
    kc, vc, ks, vs = cache.views

    def evict(out):
        return ops.evict_cache(kc, vc, weights, seqused_k=used, max_seqlen_k=n, block_table=bt, keep=keep, keep_first=2,
                               keep_last=20, k_scale_cache=ks, v_scale_cache=vs, seqused_out=out)

    new = torch.empty_like(used)
    cache.phys.copy_(raw)
    kept, _ = evict(new)
    want = (kept.clone(), cache.phys.clone(), weights.clone(), new.clone())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept_g, _ = evict(new)
    for _ in range(2):
        cache.phys.copy_(raw)
        weights.copy_(w0.transpose(1, 2))
        kept_g.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for got, ref in zip((kept_g, cache.phys, weights, new), want):
            assert torch.equal(got, ref)
    cache.phys.copy_(raw)
    weights.copy_(w0.transpose(1, 2))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        kept_s, _ = evict(new)
    side.synchronize()
    for got, ref in zip((kept_s, cache.phys, weights, new), want):
        assert torch.equal(got, ref)


def test_two_evictions_in_a_row(device):
    """A second eviction of what the first left equals the plain form applied twice."""
    n, hs, nkv, bs = 900, 128, 2, 16
    table, nblocks = U.block_tables([n], bs, seed=4)
    cache = U.Cache("int4", nblocks, bs, device, nkv=nkv, hs=hs)
    rng = np.random.default_rng(5)
    raw = rng.integers(0, 256, cache.phys.shape, dtype=np.uint8)
    cache.phys.copy_(torch.from_numpy(raw))
    w = rng.gamma(0.3, 1.0, (nblocks, bs, nkv)).astype(np.float32)
    weights = torch.from_numpy(w).to(device)
    used = torch.tensor([n], dtype=torch.int32, device=device)
    kc, vc, ks, vs = cache.views
    pages, lens = raw.transpose(0, 2, 1, 3).copy(), [n]
    for keep in (500, 123):
        kept, _ = ops.evict_cache(kc, vc, weights, seqused_k=used, max_seqlen_k=n,
                                  block_table=torch.from_numpy(table).to(device), keep=keep, keep_first=3, keep_last=40,
                                  k_scale_cache=ks, v_scale_cache=vs, seqused_out=used)
        want, lens = plain(pages, w, table, lens, keep, 3, 40, None, bs)
        torch.cuda.synchronize()
        assert np.array_equal(kept.cpu().numpy(), want) and used.tolist() == list(lens)
    assert np.array_equal(cache.phys.cpu().numpy().transpose(0, 2, 1, 3), pages)
    assert np.array_equal(weights.cpu().numpy(), w)


def test_more_tokens_than_the_selection_holds(device):
    """Above 16 x 47,104 tokens a part of the weights does not fit the cluster's shared memory and is read again."""
    check(device, "int4", 128, 1, [760001], 5000, 4, 100, seed=12)
    check(device, "int4", 128, 1, [760001, 9], 700000, 0, 0, out=True, make=ties, seed=13)
