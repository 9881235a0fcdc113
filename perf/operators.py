"""The operators that attend over a quantized paged cache and keep it small, as measured cases.

Three operators over caches in the int4_per_token_head / k8v4_per_token_head formats:
- decode: paged attention of 1 to 4 query tokens per request at head size 128 (`ops.paged_decode`);
- weights: every cached key's softmax weight, summed over the query tokens of the call and the query heads of its KV
  head, added to a paged fp32 score (`ops.accumulate_attention_weights`), from one query token to whole prompts;
- evict: the keys that stay (the first, the last and the heaviest in between) chosen per request and KV head, and
  their cells and scores moved to the front of the request's pages, here into fresh pages as a request with a shared
  prefix does it (`ops.evict_cache`).

`run` computes them in plain torch operations (own = False) or through the framework (own = True)."""
import math

import torch

own = False

BLOCK = 16          # tokens per cache page
LOG2E = 1.4426950408889634


# ------------------------------------------------------------------------------------------------------- cases


def listed():
    return [
        # the first tokens of an answer after a short prompt: launches and latency
        dict(name="decode int4 n1000 q1", op="decode", fmt="int4", dtype="bf16", hs=128, nq=32, nkv=8, seqs=1, n=1000,
             qlen=1, ragged=False),
        # one long document, one draft token
        dict(name="decode int4 n131072 q2", op="decode", fmt="int4", dtype="bf16", hs=128, nq=24, nkv=4, seqs=1,
             n=131072, qlen=2, ragged=False),
        # a serving batch of different lengths, three draft tokens, int8 keys
        dict(name="decode k8v4 b16 ragged q4", op="decode", fmt="k8v4", dtype="fp16", hs=128, nq=32, nkv=8, seqs=16,
             n=16383, qlen=4, ragged=True),
        # a full batch at long context
        dict(name="decode int4 b32 n32768 q2", op="decode", fmt="int4", dtype="bf16", hs=128, nq=24, nkv=4, seqs=32,
             n=32768, qlen=2, ragged=False),
        # scores kept up during short answers
        dict(name="weights int4 n513 q1", op="weights", fmt="int4", dtype="bf16", hs=256, nq=24, nkv=4, seqs=1, n=513,
             qlen=1, ragged=False),
        # scores kept up while one long request decodes with three draft tokens
        dict(name="weights int4 n262144 q4", op="weights", fmt="int4", dtype="bf16", hs=256, nq=24, nkv=4, seqs=1,
             n=262144, qlen=4, ragged=False),
        # scores kept up for a serving batch of different lengths
        dict(name="weights k8v4 b16 ragged q2", op="weights", fmt="k8v4", dtype="fp16", hs=128, nq=32, nkv=8, seqs=16,
             n=16383, qlen=2, ragged=True),
        # the observation window of a long prompt: its last chunk scores the whole context before a first eviction
        dict(name="weights int4 n40960 q1024", op="weights", fmt="int4", dtype="bf16", hs=256, nq=24, nkv=4, seqs=1,
             n=40960, qlen=1024, ragged=False),
        # whole prompts of different lengths, packed
        dict(name="weights k8v4 b3 whole n2777", op="weights", fmt="k8v4", dtype="bf16", hs=128, nq=32, nkv=8, seqs=3,
             n=2777, qlen=2777, ragged=True),
        # a request a little above its budget: latency
        dict(name="evict int4 n1100 keep1024", op="evict", fmt="int4", hs=128, nkv=8, seqs=1, n=1100, keep=1024,
             first=4, last=256, ragged=False),
        # one long document cut down to a budget
        dict(name="evict int4 n262143 keep32768", op="evict", fmt="int4", hs=256, nkv=4, seqs=1, n=262143, keep=32768,
             first=4, last=1000, ragged=False),
        # a serving batch cut down together
        dict(name="evict k8v4 b24 ragged keep4096", op="evict", fmt="k8v4", hs=256, nkv=4, seqs=24, n=16384, keep=4096,
             first=16, last=512, ragged=True),
    ]


def _log_int(rng, lo, hi):
    """A whole number between lo and hi, spread over the logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("decode", "weights", "evict"))
    fmt = rng.choice(("int4", "k8v4"))
    nkv = rng.choice((1, 2, 4, 8))
    seqs = _log_int(rng, 1, 32)
    ragged = rng.random() < 0.6
    if op == "decode":
        qlen = rng.randint(1, 4)
        group = rng.choice([g for g in (1, 2, 3, 4, 6, 8) if g * qlen <= 32])
        n = _log_int(rng, 1, min(131072, 4194304 // (seqs * nkv)))
        return dict(op=op, fmt=fmt, dtype=rng.choice(("bf16", "fp16")), hs=128, nq=group * nkv, nkv=nkv, seqs=seqs,
                    n=max(n, qlen), qlen=qlen, ragged=ragged)
    if op == "weights":
        hs = rng.choice((128, 256, 512))
        group = rng.choice((1, 2, 3, 4, 6, 8))
        if rng.random() < 0.5:  # decoding
            qlen = rng.randint(1, 4)
            n = _log_int(rng, 1, min(131072, 1048576 * 128 // (seqs * nkv * hs)))
        else:                   # a prompt, or the last chunk of one
            seqs = rng.randint(1, 3)
            n = _log_int(rng, 2, 20000)
            qlen = _log_int(rng, 1, min(n, 1 + 80000000 // (n * seqs * nkv * group)))
        return dict(op=op, fmt=fmt, dtype=rng.choice(("bf16", "fp16")), hs=hs, nq=group * nkv, nkv=nkv, seqs=seqs,
                    n=max(n, qlen), qlen=qlen, ragged=ragged)
    hs = rng.choice((128, 256, 512))
    n = _log_int(rng, 2, min(262144, 1048576 * 128 // (seqs * nkv * hs)))
    keep = _log_int(rng, 1, n)
    first = rng.randint(0, min(keep, 16))
    last = rng.randint(0, keep - first)
    return dict(op=op, fmt=fmt, hs=hs, nkv=nkv, seqs=seqs, n=n, keep=keep, first=first, last=last, ragged=ragged)


def _lens(case):
    """Cached tokens of every request: all n, or spread between n / 4 and n."""
    n, seqs = case["n"], case["seqs"]
    if not case["ragged"]:
        return [n] * seqs
    return [max(1, n - (i * 7919 * max(1, n // 64)) % max(1, 3 * n // 4)) for i in range(seqs)]


def _qlens(case):
    """Query tokens of every request: the last qlen of its tokens, or all of them where it has fewer."""
    return [min(case["qlen"], n) for n in _lens(case)]


def _key_bytes(case):
    return case["hs"] // 2 if case["fmt"] == "int4" else case["hs"]


def _cell(case):
    return _key_bytes(case) + 8 + case["hs"] // 2


def work(case):
    lens, nkv = _lens(case), case["nkv"]
    if case["op"] == "evict":
        kept = [min(n, case["keep"]) for n in lens]
        return {"bytes": 4 * nkv * sum(lens) + nkv * sum(kept) * (2 * _cell(case) + 4) + 4 * nkv * len(lens) * case["keep"],
                "flops": 0}
    qlens, nq, hs = _qlens(case), case["nq"], case["hs"]
    seen = sum(q * n - q * (q - 1) // 2 for q, n in zip(qlens, lens))  # (query token, key) pairs
    q_bytes = 2 * sum(qlens) * nq * hs
    if case["op"] == "decode":
        return {"bytes": nkv * _cell(case) * sum(lens) + 2 * q_bytes, "flops": 4 * seen * nq * hs}
    return {"bytes": nkv * (_key_bytes(case) + 4 + 8) * sum(lens) + q_bytes + 4 * sum(qlens) * nq,
            "flops": 2 * seen * nq * hs}


# ------------------------------------------------------------------------------------------------------ inputs


def _quantise4(x, word):
    """4-bit codes of the rows of x in pairs (low nibble = even channel) and their scale words, zero point inside."""
    mn, mx = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    scale = ((mx - mn) / 15).clamp_min(1e-6)
    zp = (-mn / scale).round().clamp(0, 15)
    u = (x / scale + zp).round().clamp(0, 15).to(torch.uint8)
    word.copy_(((scale.view(torch.int32) & -16) | zp.to(torch.int32)).view(torch.uint8))
    return u[..., 0::2] | (u[..., 1::2] << 4)


def _cache(case, blocks, gen, dev):
    """Pages (blocks, KV heads, BLOCK, cell) of keys and values as a rotated cache holds them: rows of near-normal
    channels whose magnitudes differ from token to token."""
    hs, nkv, kb = case["hs"], case["nkv"], _key_bytes(case)
    pages = torch.empty((blocks, nkv, BLOCK, _cell(case)), dtype=torch.uint8, device=dev)
    step = max(1, (1 << 26) // (nkv * BLOCK * hs))
    for b in range(0, blocks, step):
        part = pages[b:b + step]
        for is_key in (True, False):
            x = torch.randn(part.shape[:3] + (hs,), generator=gen, device=dev)
            x *= torch.exp(0.4 * torch.randn(part.shape[:3] + (1,), generator=gen, device=dev)) * math.sqrt(hs)
            if is_key and case["fmt"] == "k8v4":
                scale = (x.abs().amax(-1, keepdim=True) / 127).clamp_min(1e-6)
                part[..., :kb] = (x / scale).round().clamp(-127, 127).to(torch.int8).view(torch.uint8)
                part[..., kb:kb + 4] = scale.view(torch.uint8)
            elif is_key:
                part[..., :kb] = _quantise4(x, part[..., kb:kb + 4])
            else:
                part[..., kb + 4:kb + 4 + hs // 2] = _quantise4(x, part[..., kb + 4 + hs // 2:])
    return pages


def _views(case, pages):
    """The four views of the pages that an engine hands around: keys, values and their scales."""
    hs, kb = case["hs"], _key_bytes(case)
    blocks, nkv = pages.shape[:2]
    flat = torch.empty(0, dtype=torch.float32, device=pages.device).set_(pages.untyped_storage())
    st = [s // 4 for s in pages.stride()]
    scales = [torch.as_strided(flat, (blocks, BLOCK, nkv), (st[0], st[2], st[1]), off // 4)
              for off in (kb, kb + 4 + hs // 2)]
    if case["fmt"] == "int4":
        key, value = pages.transpose(1, 2).split(hs // 2 + 4, dim=-1)
    else:
        key = pages.view(torch.int8).transpose(1, 2)[..., :hs]
        value = pages.transpose(1, 2)[..., kb + 4:kb + 4 + hs // 2]
    return key, value, scales[0], scales[1]


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    lens = _lens(case)
    width = -(-max(lens) // BLOCK)
    wide_out = -(-case["keep"] // BLOCK) if case["op"] == "evict" else 0
    blocks = case["seqs"] * (width + wide_out) + 3
    order = torch.randperm(blocks, generator=gen, device=dev).to(torch.int32)
    table = order[:case["seqs"] * width].reshape(case["seqs"], width).contiguous()
    pages = _cache(case, blocks, gen, dev)
    key, value, k_scale, v_scale = _views(case, pages)
    state = dict(case=dict(case), pages=pages, key=key, value=value, k_scale=k_scale, v_scale=v_scale, table=table,
                 lens=torch.tensor(lens, dtype=torch.int32, device=dev))
    if case["op"] != "decode":
        # what earlier steps have summed up: heavy-tailed, none at all for a few keys
        score = torch.randn((blocks, case["nkv"], BLOCK), generator=gen, device=dev).mul_(1.5).exp_()
        score *= (torch.rand(score.shape, generator=gen, device=dev) > 0.01) / max(lens)
        state["score"] = score
        state["weights"] = score.transpose(1, 2)
    if case["op"] == "evict":
        state["out_table"] = order[case["seqs"] * width:case["seqs"] * (width + wide_out)].reshape(
            case["seqs"], wide_out).contiguous()
        return state
    dtype = torch.bfloat16 if case["dtype"] == "bf16" else torch.float16
    qlens = _qlens(case)
    cu = torch.tensor([0] + qlens, dtype=torch.int32, device=dev).cumsum(0).to(torch.int32)
    q = torch.randn((sum(qlens), case["nq"], case["hs"]), generator=gen, device=dev).to(dtype)
    state.update(q=q, cu=cu, signs=_signs(case["hs"], dev), max_q=max(qlens), max_k=max(lens),
                 scale=case["hs"] ** -0.5)
    if case["op"] == "decode":
        state["out"] = torch.empty_like(q)
    else:
        # the attention call's log-sum-exp of these rows, base 2, as it hands it to the scoring call
        state["lse"] = torch.empty((sum(qlens), case["nq"]), dtype=torch.float32, device=dev)
        group = case["nq"] // case["nkv"]
        rotated = _rotate(q.float(), state["signs"])
        for b, (ql, n) in enumerate(zip(qlens, lens)):
            at = sum(qlens[:b])
            cells = pages[table[b, :-(-n // BLOCK)].long()].transpose(0, 1).flatten(1, 2)[:, :n]
            keys = _keys(case, cells)
            for h in range(case["nkv"]):
                rows = rotated[at:at + ql, h * group:(h + 1) * group].flatten(0, 1)
                s = rows @ keys[h].T * (state["scale"] / case["hs"])
                seen = torch.arange(n, device=dev)[None] <= (n - ql + torch.arange(ql, device=dev))[:, None]
                s.masked_fill_(~seen.repeat_interleave(group, 0), -math.inf)
                state["lse"][at:at + ql, h * group:(h + 1) * group] = (
                    torch.logsumexp(s, -1) * LOG2E).reshape(ql, group)
    return state


# -------------------------------------------------------------------------------------------------- plain forms


def _signs(hs, dev):
    """The sign vector of the rotation the cache is held in: -1 where bit 63 of splitmix64(i) is set."""
    mask, out = (1 << 64) - 1, []
    for i in range(hs):
        z = (i + 0x9E3779B97F4A7C15) & mask
        z = ((z ^ (z >> 30)) * 0xBF58476D1CE4E5B9) & mask
        z = ((z ^ (z >> 27)) * 0x94D049BB133111EB) & mask
        out.append(-1.0 if (z ^ (z >> 31)) >> 63 else 1.0)
    return torch.tensor(out, dtype=torch.float32, device=dev)


def _hadamard(hs, dev, dtype=torch.float32):
    """H[i, j] = (-1)^popcount(i & j)."""
    i = torch.arange(hs, device=dev)
    x = i[:, None] & i[None]
    x = x ^ (x >> 8)
    x = x ^ (x >> 4)
    x = x ^ (x >> 2)
    x = x ^ (x >> 1)
    return (1 - 2 * (x & 1)).to(dtype)


def _rotate(x, signs):
    return (x * signs) @ _hadamard(x.shape[-1], x.device)


def _unrotate(y, signs):
    return (y @ _hadamard(y.shape[-1], y.device)) * signs / y.shape[-1]


def _codes4(cells, at, hs):
    """(u - zero point) x scale of the 4-bit rows at byte `at` of the cells, whose scale word follows them."""
    packed = cells[..., at:at + hs // 2]
    u = torch.stack((packed & 15, packed >> 4), -1).flatten(-2).float()
    word = cells[..., at + hs // 2:at + hs // 2 + 4].contiguous().view(torch.int32)
    return (u - (word & 15).float()) * (word & -16).view(torch.float32)


def _keys(case, cells):
    if case["fmt"] == "int4":
        return _codes4(cells, 0, case["hs"])
    hs = case["hs"]
    return cells[..., :hs].contiguous().view(torch.int8).float() * cells[..., hs:hs + 4].contiguous().view(torch.float32)


def _gathered(s):
    """The requests' cells (requests, KV heads, padded keys, cell), and the padded keys' positions."""
    cells = s["pages"][s["table"].long()].transpose(1, 2).flatten(2, 3)
    return cells, torch.arange(cells.shape[2], device=cells.device)


def _padded_rows(s):
    """Rotated query rows (requests, KV heads, padded query tokens, heads of the group, head size), the flat token
    each comes from, whether it exists, and the last key it sees."""
    case, dev = s["case"], s["q"].device
    seqs, nkv = case["seqs"], case["nkv"]
    cu = s["cu"].long()
    qlen = cu[1:] - cu[:-1]
    i = torch.arange(s["max_q"], device=dev)[None]
    real = i < qlen[:, None]
    token = (cu[:-1, None] + i).clamp_max(s["q"].shape[0] - 1)
    rows = _rotate(s["q"].float(), s["signs"])[token]
    rows = rows.reshape(seqs, s["max_q"], nkv, -1, case["hs"]).transpose(1, 2)
    return rows, token, real, s["lens"].long()[:, None] - qlen[:, None] + i


def _scores(s, cells, rows, visible_to, pos):
    """Scores in log2 units, -inf where a key is masked: (requests, KV heads, tokens, group, keys)."""
    case = s["case"]
    keys = _keys(case, cells)
    t = rows.flatten(2, 3) @ keys.transpose(-1, -2) * (s["scale"] / case["hs"] * LOG2E)
    t = t.reshape(rows.shape[:4] + (keys.shape[2],))
    return t.masked_fill(pos > visible_to[:, None, :, None, None], -math.inf)


def _decode_plain(s):
    case = s["case"]
    cells, pos = _gathered(s)
    rows, token, real, last = _padded_rows(s)
    t = _scores(s, cells, rows, last, pos)
    p = torch.exp2(t - t.amax(-1, keepdim=True))
    p = torch.where(pos <= last[:, None, :, None, None], p, 0.0)
    values = _codes4(cells, _key_bytes(case) + 4, case["hs"])
    values = torch.where(pos[:, None] < s["lens"][:, None, None, None], values, 0.0)
    o = (p.flatten(2, 3) @ values).reshape(rows.shape) / p.sum(-1, keepdim=True)
    o = _unrotate(o, s["signs"]).transpose(1, 2).flatten(2, 3)
    s["out"][token[real]] = o[real].to(s["out"].dtype)
    return s["out"]


def _weights_plain(s):
    cells, pos = _gathered(s)
    rows, token, real, last = _padded_rows(s)
    t = _scores(s, cells, rows, last, pos)
    lse = s["lse"][token].reshape(rows.shape[0], s["max_q"], rows.shape[1], -1).transpose(1, 2)
    t = torch.exp2(t - lse[..., None]) * real[:, None, :, None, None]
    add = t.sum((2, 3))
    # the call's own tokens have no earlier weight; every other key of a request gets its weight added
    old = s["score"][s["table"].long()].transpose(1, 2).flatten(2, 3)
    n = s["lens"].long()
    fresh = pos >= (n - (s["cu"][1:] - s["cu"][:-1]).long())[:, None]
    new = add + torch.where(fresh[:, None], 0.0, old)
    new = torch.where((pos < n[:, None])[:, None], new, old)
    s["score"][s["table"].long()] = new.unflatten(2, (-1, BLOCK)).transpose(1, 2)
    return s["weights"]


def _evict_plain(s):
    case = s["case"]
    cells, pos = _gathered(s)
    n, keep = s["lens"].long()[:, None, None], case["keep"]
    old = s["score"][s["table"].long()].transpose(1, 2).flatten(2, 3)
    stays = (pos < case["first"]) | (pos >= n - case["last"])
    rank = torch.where(stays, math.inf, old)
    rank = torch.where(pos < n, rank, -math.inf)
    order = rank.sort(dim=-1, stable=True, descending=True).indices[..., :keep]
    if order.shape[-1] < keep:
        order = torch.nn.functional.pad(order, (0, keep - order.shape[-1]), value=cells.shape[2])
    order = torch.where(order < n, order, cells.shape[2]).sort(-1).values
    real = order < cells.shape[2]
    kept = torch.where(real, order, -1).to(torch.int32)
    # the kept cells go to the front of the request's new pages, in order
    at = torch.arange(keep, device=cells.device)
    block = s["out_table"].long()[:, at // BLOCK][:, None].expand(kept.shape)[real]
    head = torch.arange(case["nkv"], device=cells.device)[None, :, None].expand(kept.shape)[real]
    slot = (at % BLOCK).expand(kept.shape)[real]
    from_ = order.clamp_max(cells.shape[2] - 1)
    s["pages"][block, head, slot] = cells.gather(2, from_[..., None].expand(from_.shape + cells.shape[3:]))[real]
    s["score"][block, head, slot] = old.gather(2, from_)[real]
    return kept, s["lens"].clamp_max(keep), s["weights"], s["pages"]


def run(s):
    case = s["case"]
    if not own:
        return {"decode": _decode_plain, "weights": _weights_plain, "evict": _evict_plain}[case["op"]](s)
    from vllm_quantpack_b200.attention import ops
    if case["op"] == "decode":
        return ops.paged_decode(s["q"], s["key"], s["value"], s["out"], cu_seqlens_q=s["cu"], max_seqlen_q=s["max_q"],
                                seqused_k=s["lens"], max_seqlen_k=s["max_k"], softmax_scale=s["scale"],
                                block_table=s["table"], k_scale_cache=s["k_scale"], v_scale_cache=s["v_scale"])
    if case["op"] == "weights":
        return ops.accumulate_attention_weights(
            s["q"], s["key"], s["value"], s["weights"], lse=s["lse"], cu_seqlens_q=s["cu"], max_seqlen_q=s["max_q"],
            seqused_k=s["lens"], max_seqlen_k=s["max_k"], softmax_scale=s["scale"], block_table=s["table"],
            k_scale_cache=s["k_scale"], v_scale_cache=s["v_scale"])
    kept, lens = ops.evict_cache(s["key"], s["value"], s["weights"], seqused_k=s["lens"], max_seqlen_k=case["n"],
                                 block_table=s["table"], keep=case["keep"], keep_first=case["first"],
                                 keep_last=case["last"], k_scale_cache=s["k_scale"], v_scale_cache=s["v_scale"],
                                 out_block_table=s["out_table"])
    return kept, lens, s["weights"], s["pages"]


# ------------------------------------------------------------------------------------------- from the definition


def _exact_rows(case, raw, at):
    """4-bit rows of raw cells (keys, cell) in 64 bits."""
    hs = case["hs"]
    word = raw[:, at + hs // 2:at + hs // 2 + 4].contiguous().view(torch.int32)
    rows = torch.empty((raw.shape[0], hs), dtype=torch.float64, device=raw.device)
    rows[:, 0::2] = (raw[:, at:at + hs // 2] % 16).double()
    rows[:, 1::2] = (raw[:, at:at + hs // 2] // 16).double()
    zp = word % 16  # the word's low four bits; the scale is the word without them
    return (rows - zp.double()) * (word - zp).view(torch.float32).double()


def exact(case, seed):
    s = prepare(case, seed)
    lens, table, pages = _lens(case), s["table"].cpu().tolist(), s["pages"]
    if case["op"] == "evict":
        # nothing is computed but the choice and the copies: the scores that the new pages hold
        score = s["score"].double()
        for b, n in enumerate(lens):
            old = score[torch.tensor(table[b], device=score.device)].transpose(0, 1).flatten(1)[:, :n].clone()
            middle = range(min(case["first"], n), max(min(case["first"], n), n - case["last"]))
            room = case["keep"] - (n - len(middle))
            for h in range(case["nkv"]):
                if n <= case["keep"]:
                    stay = list(range(n))
                else:
                    vals = old[h].cpu().tolist()
                    best = sorted(middle, key=lambda i: (-vals[i], i))[:room]
                    stay = sorted(set(range(n)) - set(middle) | set(best))
                at = torch.arange(len(stay), device=score.device)
                score[s["out_table"][b].long()[at // BLOCK], h, at % BLOCK] = old[h][torch.tensor(
                    stay, dtype=torch.long, device=score.device)]
        return None, None, score.transpose(1, 2), None
    hs, group, cu = case["hs"], case["nq"] // case["nkv"], s["cu"].cpu().tolist()
    had = _hadamard(hs, pages.device, torch.float64)
    q = (s["q"].double() * s["signs"].double()) @ had
    kb = _key_bytes(case)
    result = torch.zeros(s["q"].shape, dtype=torch.float64, device=pages.device) if case["op"] == "decode" \
        else s["score"].double()
    for b, n in enumerate(lens):
        blocks = torch.tensor(table[b][:-(-n // BLOCK)], device=pages.device)
        ql = cu[b + 1] - cu[b]
        sees = n - ql + torch.arange(ql, device=pages.device)  # last key of each query token
        hidden = (torch.arange(n, device=pages.device)[None] > sees[:, None]).repeat_interleave(group, 0)
        for h in range(case["nkv"]):
            raw = pages[blocks, h].reshape(-1, pages.shape[-1])[:n]
            if case["fmt"] == "int4":
                k = _exact_rows(case, raw, 0)
            else:
                k = raw[:, :hs].contiguous().view(torch.int8).double() * \
                    raw[:, hs:hs + 4].contiguous().view(torch.float32).double()
            rows = q[cu[b]:cu[b + 1], h * group:(h + 1) * group].reshape(-1, hs)
            t = (rows @ k.T) * (s["scale"] / hs)
            t[hidden] = -math.inf
            if case["op"] == "decode":
                o = torch.softmax(t, -1) @ _exact_rows(case, raw, kb + 4)
                o = (o @ had) * s["signs"].double() / hs
                result[cu[b]:cu[b + 1], h * group:(h + 1) * group] = o.reshape(ql, group, hs)
                continue
            lse = s["lse"][cu[b]:cu[b + 1], h * group:(h + 1) * group].double().reshape(-1, 1) * math.log(2.0)
            add = torch.exp(t - lse).sum(0)
            at = torch.arange(n, device=pages.device)
            old = result[blocks[at // BLOCK], h, at % BLOCK]
            old[n - ql:] = 0.0
            result[blocks[at // BLOCK], h, at % BLOCK] = old + add
    return result if case["op"] == "decode" else result.transpose(1, 2)
