"""B200 ops behind the plugin's patch points: cache write, split-KV decode, RHT and partial merge.

These are the functions the stock vLLM int4 module (`vllm.v1.attention.ops.int4_per_token_head`, vLLM >= 0.31)
exposes and the plugin patches (vllm_quantpack/attention/int4_kv.py:39, 212-216, 294-333;
vllm_quantpack/attention/k8v4_kv.py:152-163), with the same names, arguments and tensor views, each one a thin
launch of a CUDA kernel of libquantpack_b200.so on the current stream. There is no CPU path: on a machine without
the library or a GPU every op raises.
"""
import threading

import torch

from .. import _lib
from . import rht

_DTYPES = {torch.bfloat16: 0, torch.float16: 1}
FMT_INT4, FMT_K8V4 = 0, 1
MAX_Q_DECODE_ROWS = 32      # query rows (tokens x query heads per KV head) one decode CTA holds


def _stream(device):
    """The current stream's handle (of an indexed device without building the stream object: every op asks twice)."""
    if type(device) is torch.device and device.index is not None:
        return torch._C._cuda_getCurrentRawStream(device.index)
    return torch.cuda.current_stream(device).cuda_stream


def _device_key(device):
    return device if type(device) is torch.device else torch.device(device)


def _sinks_ptr(sinks, nq, mode):
    """Device pointer of fp32 sink logits (one per query head), or None. Sinks count once in a row's softmax, so
    only the model-domain output (mode 0) can take them, never a partial."""
    if sinks is None:
        return None
    if mode != 0:
        raise ValueError("sinks apply to the model-domain output only, not to partials")
    if sinks.dim() != 1 or sinks.shape[0] != nq:
        raise ValueError(f"sinks must have one logit per query head ({nq}), got {tuple(sinks.shape)}")
    if sinks.dtype != torch.float32 or not sinks.is_contiguous():
        # a temporary on the current stream: torch's caching allocator hands its memory to a later allocation only
        # in stream order, after the merge kernel that reads it
        sinks = sinks.float().contiguous()
    return sinks.data_ptr()


def _lse_ptr(lse_out, rows, nq, mode, out_fp32_lse):
    """Device pointer of `lse_out` ((tokens, query heads) fp32, base-2 log-sum-exp beside a model-domain output)."""
    if lse_out is None:
        return None
    if mode != 0 or out_fp32_lse is not None:
        raise ValueError("lse_out goes with the model-domain output (a partial's lse is out_fp32_lse)")
    if lse_out.dtype != torch.float32 or tuple(lse_out.shape) != (rows, nq) or not lse_out.is_contiguous():
        raise ValueError(f"lse_out must be contiguous fp32 ({rows}, {nq})")
    return lse_out.data_ptr()


def _check_device(device, **tensors):
    """The launch goes to the current device: every tensor given has to live there (a kernel that is handed another
    device's address, or the host's, faults)."""
    index = device.index
    if index is None:
        raise ValueError(f"the tensors are on {device}, the kernels run on the current device, a GPU")
    if index != torch.cuda.current_device():
        raise ValueError(f"the tensors are on {device}, the current device is {torch.cuda.current_device()}")
    for name, t in tensors.items():
        if t is not None and t.get_device() != index:
            raise ValueError(f"{name} is on {t.device}, expected {device}")


def _dtype_code(t, what):
    code = _DTYPES.get(t.dtype)
    if code is None:
        raise TypeError(f"{what}: dtype {t.dtype} (bf16 or fp16 expected)")
    return code


class CacheLayout:
    """Byte layout of a paged int4 / k8v4 cache, derived from the four views vLLM passes (`of` keeps the layouts it
    derived, keyed by everything they are derived from, so a call on the same cache pays for the checks once).

    int4 views (tests/test_int4_kv.py:95-103): key / value (blocks, block size, KV heads, hs/2 + 4) uint8 over cells
    [K | K scale | V | V scale]; k8v4 views (vllm_quantpack/attention/k8v4_kv.py:41-65): key (..., hs) int8, value
    (..., hs/2) uint8. Scale views are fp32 (blocks, block size, KV heads) over the same storage."""

    def __init__(self, k_cache, v_cache, k_scale_cache, v_scale_cache, head_size):
        if k_cache.dtype == torch.int8:
            self.fmt, kb = FMT_K8V4, head_size
        elif k_cache.dtype == torch.uint8:
            self.fmt, kb = FMT_INT4, head_size // 2
        else:
            raise TypeError(f"key cache dtype {k_cache.dtype}: uint8 (int4) or int8 (k8v4) expected")
        if k_cache.dim() != 4 or v_cache.dim() != 4:
            raise ValueError("cache views must be (blocks, block size, KV heads, bytes)")
        self.nblocks, self.block_size, self.nkv = k_cache.shape[0], k_cache.shape[1], k_cache.shape[2]
        self.head_size = head_size
        base = k_cache.data_ptr()
        self.base = base
        self.block_stride, self.slot_stride, self.head_stride = (int(s) for s in k_cache.stride()[:3])
        self.k_off = 0
        self.ks_off = k_scale_cache.data_ptr() - base
        self.v_off = v_cache.data_ptr() - base
        self.vs_off = v_scale_cache.data_ptr() - base
        self.cell = kb + 8 + head_size // 2
        if (tuple(v_cache.stride()[:3]) != (self.block_stride, self.slot_stride, self.head_stride)
                or tuple(v_cache.shape[:3]) != tuple(k_cache.shape[:3])):
            raise ValueError("key and value cache views disagree on blocks / slots / heads")
        for sc in (k_scale_cache, v_scale_cache):
            if sc.dtype != torch.float32 or tuple(sc.shape) != (self.nblocks, self.block_size, self.nkv):
                raise ValueError("scale views must be fp32 (blocks, block size, KV heads)")
            if tuple(4 * s for s in sc.stride()) != (self.block_stride, self.slot_stride, self.head_stride):
                raise ValueError("scale views must share the cache's strides")
        if self.ks_off != kb or self.v_off != kb + 4 or self.vs_off != kb + 4 + head_size // 2:
            raise ValueError(f"cell fields at K 0, K scale {self.ks_off}, V {self.v_off}, V scale {self.vs_off}: "
                             f"expected 0, {kb}, {kb + 4}, {kb + 4 + head_size // 2}")

    _known = {}

    @classmethod
    def of(cls, k_cache, v_cache, k_scale_cache, v_scale_cache, head_size):
        """The layout of these views: a derived one when every input to the derivation (addresses, dtypes, shapes,
        strides, head size) matches, else a new one (checked; only valid layouts are kept)."""
        key = (k_cache.data_ptr(), v_cache.data_ptr(), k_scale_cache.data_ptr(), v_scale_cache.data_ptr(),
               k_cache.dtype, v_cache.dtype, k_scale_cache.dtype, v_scale_cache.dtype, k_cache.shape, v_cache.shape,
               k_scale_cache.shape, v_scale_cache.shape, k_cache.stride(), v_cache.stride(), k_scale_cache.stride(),
               v_scale_cache.stride(), head_size)
        lay = cls._known.get(key)
        if lay is None:
            lay = cls(k_cache, v_cache, k_scale_cache, v_scale_cache, head_size)
            if len(cls._known) >= 256:
                cls._known.clear()
            cls._known[key] = lay
        return lay

    def args(self):
        return (self.base, self.block_size, self.block_stride, self.head_stride, self.slot_stride, self.k_off,
                self.ks_off, self.v_off, self.vs_off)

    @property
    def hnd(self):
        return self.slot_stride == self.cell


# ------------------------------------------------------------------------------------------------------ RHT


def single_rht(x, inverse=False):
    """Randomized Hadamard transform over the last axis of fp32 `x` (unnormalised; see rht.py). Returns fp32."""
    if x.dtype != torch.float32:
        raise TypeError("single_rht takes fp32 (as the callers pass x.float())")
    hs = x.shape[-1]
    xc = x.contiguous()
    y = torch.empty_like(xc)
    rows = xc.numel() // hs if hs else 0
    _lib.call("qp_single_rht", xc.data_ptr(), y.data_ptr(), rows, hs, int(bool(inverse)),
              rht.device_sign_bits(hs, x.device).data_ptr(), _stream(x.device))
    return y


# ------------------------------------------------------------------------------------------------------ cache write


def reshape_and_cache_int4(key, value, key_cache, value_cache, slot_mapping, *, k_scale_cache, v_scale_cache,
                           rotate=True):
    """Rotate, quantize and write key / value (tokens, KV heads, hs) into the cache; slots < 0 are skipped.
    A uint8 key view is the int4 cache, an int8 one k8v4 (vllm_quantpack/attention/k8v4_kv.py:36-38, 152-157).
    rotate=False takes key / value as already in the RHT domain (the `_store_k8v4` kernel contract)."""
    hs = key.shape[-1]
    if value.shape[-1] != hs:
        raise ValueError(f"key head size {hs} != value head size {value.shape[-1]}")
    if key.stride(-1) != 1 or value.stride(-1) != 1:
        raise ValueError("key / value rows must be contiguous")
    lay = CacheLayout.of(key_cache, value_cache, k_scale_cache, v_scale_cache, hs)
    if slot_mapping.dtype != torch.int64:
        slot_mapping = slot_mapping.to(torch.int64)
    slot_mapping = slot_mapping.contiguous()
    dt = _dtype_code(key, "reshape_and_cache_int4")
    if value.dtype != key.dtype:
        raise TypeError("key and value dtypes differ")
    name = "qp_reshape_and_cache_int4" if lay.fmt == FMT_INT4 else "qp_reshape_and_cache_k8v4"
    _lib.call(name, key.data_ptr(), value.data_ptr(), dt, key.shape[0], key.shape[1], hs, key.stride(0),
              key.stride(1), value.stride(0), value.stride(1), slot_mapping.data_ptr(), *lay.args(),
              rht.device_sign_bits(hs, key.device).data_ptr(), int(bool(rotate)), _stream(key.device))


# ------------------------------------------------------------------------------------------------------ decode

_ws_lock = threading.Lock()
_workspaces = {}


_retired = []


def workspace(device, nbytes):
    """A scratch buffer for the split-KV partials, grown geometrically and kept for the process: the device's own for
    calls on the default stream and those captured into a graph, one more for every other stream with eager calls (calls
    on two streams may overlap). A buffer that is outgrown stays allocated too: a CUDA graph captured earlier may still
    hold its address. Growing it inside a CUDA-graph capture allocates from the graph's pool: reserve the largest size
    before capturing (`reserve_workspace`)."""
    stream = _stream(device)
    if stream and torch.cuda.is_current_stream_capturing():
        stream = 0
    return _workspace(_device_key(device), stream, nbytes)


def reserve_workspace(device, nbytes):
    """Grows the device's own buffer, whatever the current stream: what captured calls use."""
    return _workspace(_device_key(device), 0, nbytes)


def _workspace(device, stream, nbytes):
    key = (device, stream)
    ws = _workspaces.get(key)
    if ws is not None and ws.numel() >= nbytes:  # the common case: no growth, no lock
        return ws
    with _ws_lock:
        ws = _workspaces.get(key)
        if ws is None or ws.numel() < nbytes:
            if ws is not None:
                _retired.append(ws)
            size = max(nbytes, 2 * (ws.numel() if ws is not None else 0), 1 << 20)
            ws = torch.empty(size, dtype=torch.uint8, device=device)
            _workspaces[key] = ws
    return ws


_sm_counts = {}


def sm_count(device):
    key = _device_key(device)
    n = _sm_counts.get(key)
    if n is None:
        n = _sm_counts[key] = torch.cuda.get_device_properties(device).multi_processor_count
    return n


VARLEN_MAX_Q = 32   # query tokens of a varlen sub-sequence at most (32 query rows per KV head)


def window_keys(max_seqlen_k, sliding_window, max_q):
    """Keys the split count is sized for: the context, or with a sliding window the span of the tiles a request's
    windows cover (its first token's window start to its last token, plus a partial tile)."""
    max_seqlen_k = int(max_seqlen_k)
    if sliding_window and sliding_window > 0:
        return min(max_seqlen_k, int(sliding_window) + int(max_q) - 1 + 127)
    return max_seqlen_k


_sizes = {}   # host-side size arithmetic of the library, by its arguments


def _memo(fn_name, *args):
    key = (fn_name,) + args
    v = _sizes.get(key)
    if v is None:
        if len(_sizes) >= 4096:
            _sizes.clear()
        v = _sizes[key] = getattr(_lib.load(), fn_name)(*args)
    return v


def decode_num_splits(num_seqs, num_kv_heads, max_seqlen_k, sms):
    return _memo("qp_decode_num_splits", int(num_seqs), int(num_kv_heads), int(max_seqlen_k), int(sms))


def paged_decode(q, key_cache, value_cache, out, *, cu_seqlens_q, max_seqlen_q, seqused_k, max_seqlen_k,
                 softmax_scale, block_table, k_scale_cache, v_scale_cache, num_splits=None, q_rotated=False,
                 out_fp32_lse=None, ws=None, partials_only=False, tokens_after_keys=0, sliding_window=0,
                 softcap=0.0, sinks=None, lse_out=None):
    """Split-KV decode of up to 32 query rows per KV head (4 MTP tokens x 6 heads) over the paged cache.

    q / out (tokens, query heads, hs); block_table (sequences, pages), or a single sequence's row. When `out_fp32_lse`
    is a tensor (tokens, query heads) fp32, `out` must be fp32 and receives the RHT-domain output with its base-2
    log-sum-exp in `out_fp32_lse` (the partial a sequence-parallel rank exchanges); otherwise `out` gets the
    model-domain output in q's dtype. partials_only=True launches the split kernel alone and leaves its partials in the
    workspace (returned). tokens_after_keys: sequence tokens that follow
    the cached keys given here (a sequence-parallel rank holding an earlier range): query token i of a sequence sees
    key k iff k <= seqused_k - qlen + i + tokens_after_keys. sliding_window: vLLM's SLIDING_WINDOW (1 +
    window_size[0], 0 = none): that token then sees only the keys k > its last key - sliding_window. softcap > 0:
    vLLM's logit softcap, every score S becomes softcap * tanh(S / softcap). sinks: None or (query heads,) sink
    logits whose exp joins every row's softmax denominator (vLLM's attention sinks; model-domain output only).
    lse_out: None or (tokens, query heads) fp32, filled with the base-2 log-sum-exp of each row's scaled scores, sinks
    included (what `accumulate_attention_weights` takes), beside a model-domain output."""
    tokens, nq, hs = q.shape
    q_st, q_sh, q_sc = q.stride()
    out_st, out_sh, out_sc = out.stride()
    device = q.device
    lay = CacheLayout.of(key_cache, value_cache, k_scale_cache, v_scale_cache, hs)
    nkv = lay.nkv
    num_seqs = cu_seqlens_q.shape[0] - 1
    _check_device(device, key_cache=key_cache, out=out, cu_seqlens_q=cu_seqlens_q, seqused_k=seqused_k,
                  block_table=block_table, sinks=sinks, lse_out=lse_out, out_fp32_lse=out_fp32_lse, ws=ws)
    if num_splits is None:
        keys = window_keys(max_seqlen_k, sliding_window, max_seqlen_q)
        if hs == 128:
            num_splits = _memo("qp_decode_num_splits_head", hs, int(max_seqlen_q) * (nq // nkv), num_seqs, nkv, keys,
                               sm_count(device))
        else:
            num_splits = decode_num_splits(num_seqs, nkv, keys, sm_count(device))
    wbytes = _memo("qp_decode_workspace_bytes", tokens, nq, hs, int(num_splits))
    if ws is None:
        ws = workspace(device, wbytes)
    int32, bt_st = torch.int32, block_table.stride()
    if (cu_seqlens_q.dtype != int32 or seqused_k.dtype != int32 or block_table.dtype != int32
            or cu_seqlens_q.stride(0) != 1 or seqused_k.stride(0) != 1 or bt_st[-1] != 1):
        _check_index(cu_seqlens_q=cu_seqlens_q, seqused_k=seqused_k, block_table=block_table)   # names the one
    if len(bt_st) == 1 and num_seqs > 1:
        raise ValueError(f"a one-dimensional block_table serves one sequence, not {num_seqs}")
    if q_sc != 1 or out_sc != 1:
        raise ValueError("q / out rows must be contiguous")
    dt = _dtype_code(q, "paged_decode")
    if partials_only:
        mode, lse_ptr = 2, None
    elif out_fp32_lse is not None:
        if out.dtype != torch.float32 or out_fp32_lse.dtype != torch.float32:
            raise TypeError("out and lse must be fp32 for the RHT-domain output")
        if not out_fp32_lse.is_contiguous():
            raise ValueError("lse must be contiguous (tokens, query heads)")
        mode, lse_ptr = 1, out_fp32_lse.data_ptr()
    else:
        if out.dtype != q.dtype:
            raise TypeError("out dtype must match q")
        mode, lse_ptr = 0, None
    if lse_out is not None:
        lse_ptr = _lse_ptr(lse_out, tokens, nq, mode, out_fp32_lse)
    _lib.call("qp_paged_decode", lay.fmt, dt, q.data_ptr(), q_st, q_sh, out.data_ptr(), out_st, out_sh, tokens,
              num_seqs, cu_seqlens_q.data_ptr(), seqused_k.data_ptr(), int(max_seqlen_q), block_table.data_ptr(), bt_st[0],
              *lay.args(), nq, nkv, hs, float(softmax_scale), rht.device_sign_bits(hs, device).data_ptr(),
              int(bool(q_rotated)), int(tokens_after_keys), int(sliding_window), float(softcap or 0.0),
              _sinks_ptr(sinks, nq, mode), mode, lse_ptr, int(num_splits), ws.data_ptr(), ws.nbytes, _stream(device))
    return ws if partials_only else out


def merge_attn_partials(part_o, part_lse, out, lse_out=None):
    """Fold P partials part_o (P, tokens, heads, hs) fp32 / part_lse (P, tokens, heads) base-2 into `out`: in the
    model domain (inverse RHT / head, out's dtype) or, with `lse_out`, fp32 in the RHT domain plus the folded lse."""
    P, T, H, hs = part_o.shape
    if part_o.dtype != torch.float32 or part_lse.dtype != torch.float32:
        raise TypeError("partials must be fp32")
    if part_o.stride(-1) != 1:
        raise ValueError("partial rows must be contiguous")
    if lse_out is not None:
        if out.dtype != torch.float32 or not lse_out.is_contiguous():
            raise TypeError("out must be fp32 and lse_out contiguous")
        mode, dt, lptr, sbits = 1, 0, lse_out.data_ptr(), None
    else:
        mode, dt, lptr = 0, _dtype_code(out, "merge_attn_partials"), None
        sbits = rht.device_sign_bits(hs, out.device).data_ptr()
    _lib.call("qp_merge_attn_partials", dt, hs, T, H, P, part_o.data_ptr(), part_o.stride(1), part_o.stride(2),
              part_o.stride(0), part_lse.data_ptr(), part_lse.stride(1), part_lse.stride(2), part_lse.stride(0), mode,
              out.data_ptr(), out.stride(0), out.stride(1), lptr, sbits, _stream(out.device))
    return out


def fold_peer_partials(bases, rank, world, epoch, num_tokens, num_heads, head_size, out, lse_out=None):
    """Rank fold over NVLink (qp_fold_peer_partials): `bases` an int64 device tensor of the ranks' exchange buffer
    addresses, every rank's partial of call `epoch` already in its own buffer."""
    if lse_out is not None:
        if out.dtype != torch.float32 or not lse_out.is_contiguous():
            raise TypeError("out must be fp32 and lse_out contiguous")
        mode, dt, lptr, sbits = 1, 0, lse_out.data_ptr(), None
    else:
        mode, dt, lptr = 0, _dtype_code(out, "fold_peer_partials"), None
        sbits = rht.device_sign_bits(head_size, out.device).data_ptr()
    if out.stride(-1) != 1:
        raise ValueError("out rows must be contiguous")
    _lib.call("qp_fold_peer_partials", dt, head_size, num_tokens, num_heads, world, rank, bases.data_ptr(),
              epoch & 0xFFFFFFFF, mode, out.data_ptr(), out.stride(0), out.stride(1), lptr, sbits, _stream(out.device))
    return out


# ------------------------------------------------------------------------------------------------------ prefill


def prefill(q, key_cache, value_cache, out, *, block_row, n, softmax_scale, k_scale_cache, v_scale_cache,
            q_rotated=False, out_fp32_lse=None, ws=None, tokens_after_keys=0, lse_out=None):
    """Chunk prefill of one sequence on the tensor cores: q (qlen, query heads, hs) are the last qlen positions of a
    context of n cached tokens (causal among themselves); block_row is the sequence's int32 block-table row.
    `out` gets the model-domain output in q's dtype, or with `out_fp32_lse` the fp32 RHT-domain output and its
    base-2 lse (vllm_quantpack/attention/int4_prefill.py:203-232 returns the RHT-domain output for rotated queries).
    tokens_after_keys (n >= qlen - tokens_after_keys) and lse_out as in paged_decode."""
    hs, nq, qlen = q.shape[-1], q.shape[1], q.shape[0]
    lay = CacheLayout.of(key_cache, value_cache, k_scale_cache, v_scale_cache, hs)
    if block_row.dtype != torch.int32 or block_row.stride(-1) != 1:
        raise TypeError("block_row must be a contiguous int32 row")
    if q.stride(-1) != 1 or out.stride(-1) != 1:
        raise ValueError("q / out rows must be contiguous")
    dt = _dtype_code(q, "prefill")
    _check_device(q.device, key_cache=key_cache, out=out, block_row=block_row, lse_out=lse_out,
                  out_fp32_lse=out_fp32_lse, ws=ws)
    wbytes = _lib.load().qp_prefill_workspace_bytes(qlen, int(n), nq, lay.nkv, hs, int(tokens_after_keys))
    if ws is None:
        ws = workspace(q.device, wbytes)
    if out_fp32_lse is not None:
        if out.dtype != torch.float32 or out_fp32_lse.dtype != torch.float32 or not out_fp32_lse.is_contiguous():
            raise TypeError("out and lse must be fp32 (lse contiguous) for the RHT-domain output")
        mode, lse_ptr = 1, out_fp32_lse.data_ptr()
    else:
        if out.dtype != q.dtype:
            raise TypeError("out dtype must match q")
        mode, lse_ptr = 0, None
    lse_ptr = _lse_ptr(lse_out, qlen, nq, mode, out_fp32_lse) or lse_ptr
    _lib.call("qp_prefill", lay.fmt, dt, q.data_ptr(), q.stride(0), q.stride(1), out.data_ptr(), out.stride(0),
              out.stride(1), qlen, int(n), block_row.data_ptr(), *lay.args(), nq, lay.nkv, hs, float(softmax_scale),
              rht.device_sign_bits(hs, q.device).data_ptr(), int(bool(q_rotated)), int(tokens_after_keys), mode,
              lse_ptr, ws.data_ptr(), ws.numel() * ws.element_size(), _stream(q.device))
    return out


def prefill_varlen(q, key_cache, value_cache, out, *, cu_seqlens_q, seqused_k, max_seqlen_k, block_table,
                   softmax_scale, k_scale_cache, v_scale_cache, q_rotated=False, out_fp32_lse=None, ws=None,
                   sliding_window=0, softcap=0.0, sinks=None, lse_out=None):
    """Several short prefill chunks in ONE launch (the reference's Triton sub-batch of the chunks that are not long,
    vllm_quantpack/attention/int4_kv.py:313-323): request i's query tokens q[cu_seqlens_q[i]:cu_seqlens_q[i + 1]] are
    the last positions of its context of seqused_k[i] cached tokens, causal among themselves, read through
    block_table[i]. Split on the device into sub-sequences of 32 / group tokens for the split-KV kernel, so nothing
    is read back to the host; max_seqlen_k (a host int, an upper bound of seqused_k) sizes the split count.
    `out` as in prefill; sliding_window, softcap, sinks and lse_out as in paged_decode."""
    hs, nq, T = q.shape[-1], q.shape[1], q.shape[0]
    lay = CacheLayout.of(key_cache, value_cache, k_scale_cache, v_scale_cache, hs)
    for name, t in (("cu_seqlens_q", cu_seqlens_q), ("seqused_k", seqused_k), ("block_table", block_table)):
        if t.dtype != torch.int32 or t.stride(-1) != 1:
            raise TypeError(f"{name} must be int32 with contiguous rows")
    if q.stride(-1) != 1 or out.stride(-1) != 1:
        raise ValueError("q / out rows must be contiguous")
    dt = _dtype_code(q, "prefill_varlen")
    _check_device(q.device, key_cache=key_cache, out=out, cu_seqlens_q=cu_seqlens_q, seqused_k=seqused_k,
                  block_table=block_table, sinks=sinks, lse_out=lse_out, out_fp32_lse=out_fp32_lse, ws=ws)
    chunks = seqused_k.shape[0]
    lib = _lib.load()
    max_k = window_keys(max_seqlen_k, sliding_window, VARLEN_MAX_Q)
    wbytes = lib.qp_prefill_varlen_workspace_bytes(T, chunks, nq, lay.nkv, hs, max_k)
    if ws is None:
        ws = workspace(q.device, wbytes)
    if out_fp32_lse is not None:
        if out.dtype != torch.float32 or out_fp32_lse.dtype != torch.float32 or not out_fp32_lse.is_contiguous():
            raise TypeError("out and lse must be fp32 (lse contiguous) for the RHT-domain output")
        mode, lse_ptr = 1, out_fp32_lse.data_ptr()
    else:
        if out.dtype != q.dtype:
            raise TypeError("out dtype must match q")
        mode, lse_ptr = 0, None
    lse_ptr = _lse_ptr(lse_out, T, nq, mode, out_fp32_lse) or lse_ptr
    _lib.call("qp_prefill_varlen", lay.fmt, dt, q.data_ptr(), q.stride(0), q.stride(1), out.data_ptr(),
              out.stride(0), out.stride(1), T, chunks, cu_seqlens_q.data_ptr(), seqused_k.data_ptr(),
              max_k, block_table.data_ptr(), block_table.stride(0), *lay.args(), nq, lay.nkv, hs,
              float(softmax_scale), rht.device_sign_bits(hs, q.device).data_ptr(), int(bool(q_rotated)),
              int(sliding_window), float(softcap or 0.0), _sinks_ptr(sinks, nq, mode), mode, lse_ptr, ws.data_ptr(),
              ws.numel() * ws.element_size(), _stream(q.device))
    return out


# ------------------------------------------------------------------------------------------------------ eviction


def new_attention_weights(k_scale_cache):
    """Zeroed attention weights for a cache: fp32 (blocks, block size, KV heads) as the cache's scale views, each
    page's weights of a KV head contiguous."""
    nblocks, block_size, nkv = k_scale_cache.shape
    return torch.zeros((nblocks, nkv, block_size), dtype=torch.float32, device=k_scale_cache.device).transpose(1, 2)


def _check_weights(weights, lay):
    if weights.dtype != torch.float32 or weights.shape != (lay.nblocks, lay.block_size, lay.nkv):
        raise ValueError(f"weights must be fp32 (blocks, block size, KV heads) = "
                         f"({lay.nblocks}, {lay.block_size}, {lay.nkv}), got {weights.dtype} {tuple(weights.shape)}")


def _check_index(**tensors):
    for name, t in tensors.items():
        if t.dtype != torch.int32:
            raise TypeError(f"{name} must be int32")
        if t.stride(-1) != 1:
            raise ValueError(f"{name} rows must be contiguous")


def _check_table(name, table, num_seqs, tokens, block_size):
    """A row of pages for every sequence, wide enough for `tokens` (one sequence's may come without the sequence axis)."""
    rows = table.shape[0] if table.dim() > 1 else 1
    if num_seqs > 0 and (rows < num_seqs or table.shape[-1] * block_size < tokens):
        raise ValueError(f"{name} {tuple(table.shape)} needs pages of {block_size} for {tokens} tokens of each of "
                         f"{num_seqs} sequences")


def accumulate_attention_weights(q, key_cache, value_cache, weights, *, lse, cu_seqlens_q, max_seqlen_q, seqused_k,
                                 max_seqlen_k, softmax_scale, block_table, k_scale_cache, v_scale_cache,
                                 q_rotated=False, ws=None, tokens_after_keys=0, sliding_window=0, softcap=0.0):
    """Add to `weights` (fp32 (blocks, block size, KV heads), `new_attention_weights`) the softmax weight that every
    cached key gets from the query rows of an attention call: q, the lengths, the block table, the scale and the
    layer's features as that call took them, `lse` the (tokens, query heads) base-2 log-sum-exp it returned in its
    `lse_out`. Summed over the query tokens (one, or a whole prompt) and the query heads of each KV head. The call's own
    tokens have no earlier weight: theirs is stored, so pages need no clearing before reuse as long as every token
    enters through such a call; a first call that covers only the last tokens of a prompt wants the other cells zeroed.
    Cells past a sequence's length are left as they are. max_seqlen_k bounds the lengths, and block_table has pages for as
    many tokens. Eager calls on two streams may overlap; graphs that are replayed at once, or beside eager calls on the
    default stream, need workspaces of their own (`ws`). Returns `weights`."""
    tokens, nq, hs = q.shape
    q_st, q_sh, q_sc = q.stride()
    lay = CacheLayout.of(key_cache, value_cache, k_scale_cache, v_scale_cache, hs)
    _check_weights(weights, lay)
    _check_index(cu_seqlens_q=cu_seqlens_q, seqused_k=seqused_k, block_table=block_table)
    if q_sc != 1:
        raise ValueError("q rows must be contiguous")
    if lse.dtype != torch.float32 or lse.shape != (tokens, nq) or not lse.is_contiguous():
        raise ValueError(f"lse must be contiguous fp32 ({tokens}, {nq})")
    dt = _dtype_code(q, "accumulate_attention_weights")
    _check_device(q.device, key_cache=key_cache, weights=weights, lse=lse, cu_seqlens_q=cu_seqlens_q,
                  seqused_k=seqused_k, block_table=block_table, ws=ws)
    num_seqs = cu_seqlens_q.shape[0] - 1
    if seqused_k.shape[0] < num_seqs:
        raise ValueError(f"seqused_k has {seqused_k.shape[0]} lengths for {num_seqs} sequences")
    _check_table("block_table", block_table, num_seqs, int(max_seqlen_k), lay.block_size)
    if ws is None:
        ws = workspace(q.device, _memo("qp_attn_weights_workspace_bytes", tokens, num_seqs, int(max_seqlen_q), nq,
                                       lay.nkv, hs))
    _lib.call("qp_accumulate_attn_weights", lay.fmt, dt, q.data_ptr(), q_st, q_sh, tokens, num_seqs,
              cu_seqlens_q.data_ptr(), seqused_k.data_ptr(), int(max_seqlen_q), int(max_seqlen_k),
              block_table.data_ptr(), block_table.stride(0), *lay.args(), nq, lay.nkv, hs, float(softmax_scale),
              rht.device_sign_bits(hs, q.device).data_ptr(), int(bool(q_rotated)), int(tokens_after_keys),
              int(sliding_window), float(softcap or 0.0), lse.data_ptr(), weights.data_ptr(), *weights.stride(),
              ws.data_ptr(), ws.nbytes, _stream(q.device))
    return weights


def evict_cache(key_cache, value_cache, weights, *, seqused_k, max_seqlen_k, block_table, keep, keep_first=0,
                keep_last=0, k_scale_cache, v_scale_cache, out_block_table=None, seqused_out=None, ws=None):
    """Cut every sequence of more than `keep` cached tokens down to `keep`: per KV head its first `keep_first` tokens,
    its last `keep_last` and the heaviest by `weights` in between (of equal ones the earlier). The kept cells and
    weights move to the front of the sequence's pages, in their order, so each KV head may keep other tokens and the
    sequence stays a sequence of min(length, keep) tokens for every call that reads it. In place (no other sequence may
    hold the pages), or with `out_block_table` (int32 (seqs, pages)) into other pages, the old ones left as they are: a
    sequence whose pages others share (a common prompt). Returns (kept, seqused): the old positions (seqs, KV heads,
    keep) int32, -1 behind the last, and the new lengths (`seqused_out` if given, which may be `seqused_k` itself).
    max_seqlen_k bounds the lengths, and block_table has pages for as many tokens.
    Workspaces (`ws`) as for `accumulate_attention_weights`."""
    int4 = key_cache.dtype == torch.uint8
    hs = (key_cache.shape[-1] - 4) * 2 if int4 else key_cache.shape[-1]
    lay = CacheLayout.of(key_cache, value_cache, k_scale_cache, v_scale_cache, hs)
    _check_weights(weights, lay)
    _check_index(seqused_k=seqused_k, block_table=block_table)
    num_seqs, keep = seqused_k.shape[0], int(keep)
    _check_table("block_table", block_table, num_seqs, int(max_seqlen_k), lay.block_size)
    if out_block_table is not None:
        _check_index(out_block_table=out_block_table)
        _check_table("out_block_table", out_block_table, num_seqs, min(keep, int(max_seqlen_k)), lay.block_size)
    if seqused_out is None:
        seqused_out = torch.empty_like(seqused_k)
    elif seqused_out.dtype != torch.int32 or seqused_out.shape != seqused_k.shape or not seqused_out.is_contiguous():
        raise ValueError("seqused_out must be contiguous int32, one length per sequence")
    _check_device(key_cache.device, weights=weights, seqused_k=seqused_k, block_table=block_table,
                  seqused_out=seqused_out, out_block_table=out_block_table, ws=ws)
    kept = torch.empty((num_seqs, lay.nkv, max(keep, 0)), dtype=torch.int32, device=key_cache.device)
    if ws is None:
        ws = workspace(key_cache.device, _memo("qp_evict_workspace_bytes", num_seqs, lay.nkv, int(max_seqlen_k), keep))
    _lib.call("qp_evict_cache", lay.base, lay.cell, lay.block_size, lay.block_stride, lay.head_stride, lay.slot_stride,
              lay.nkv, weights.data_ptr(), *weights.stride(), num_seqs, seqused_k.data_ptr(), int(max_seqlen_k),
              block_table.data_ptr(), block_table.stride(0),
              out_block_table.data_ptr() if out_block_table is not None else None,
              out_block_table.stride(0) if out_block_table is not None else 0, keep, int(keep_first), int(keep_last),
              kept.data_ptr(), seqused_out.data_ptr(), ws.data_ptr(), ws.nbytes,
              _stream(key_cache.device))
    return kept, seqused_out
