"""Serving operators of a decoder: a paged key-value cache and the attention on it.

    kv_append         rotate new keys (and queries) by their positions, write
                      keys and values to their slots of a paged cache
    prompt_attention  (causal) attention over packed prompts, grouped heads
    paged_decode      attention of one new token per sequence over its cache

They work on torch CUDA tensors (f16 or bf16, sums in f32), run on the current
stream of the tensors' device, allocate nothing but their outputs and a
workspace per stream, wait for nothing and can be captured into a CUDA graph.
A cache is any pair of tensors [pages, page_size, kv_heads, dim] whose head
vectors are contiguous and start on 16-byte boundaries; a page may be stored
token by token or head by head (a transposed view).  Index tensors are int32.

Arguments of a wrong shape or type raise ValueError, forms that the kernels do
not take NotImplementedError.  Indices are data on the device: one out of its
range touches no memory and is reported by ``check_status``.  (The reference
has no such operators; its paged attention example,
examples/triton-ktir/paged_attention.mlir, runs through KTIRInterpreter.)
"""

from __future__ import annotations

import ctypes as C

import torch

from . import runtime as R

_DTYPES = {torch.float16: R.F16, torch.bfloat16: R.BF16}
_STATUS = {}
_WORKSPACES = {}


def _status(device):
    t = _STATUS.get(device)
    if t is None:
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("call a serving operator once on this device before capturing it")
        t = _STATUS[device] = torch.zeros(1, dtype=torch.int32, device=device)
        torch.cuda.synchronize(device)   # whichever stream asks for it next sees it cleared
    return t


def check_status(device=None) -> None:
    """Wait for `device` (default: the current one) and raise for what the
    serving operators have reported there since the last check."""
    device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    if device.index is None:
        device = torch.device("cuda", torch.cuda.current_device())
    t = _STATUS.get(device)
    if t is None:
        return
    torch.cuda.synchronize(device)
    v = int(t.item())
    if v:
        t.zero_()
        torch.cuda.synchronize(device)
    if v & R.STATUS_BAD_INDEX:
        raise IndexError("a page, slot, position, length or offset of a serving operator is out of range")
    if v & R.STATUS_TIMEOUT:
        raise RuntimeError("device wait timed out")


def _workspace(nbytes, device, stream):
    """Zeroed scratch of at least `nbytes` for calls on `stream`, kept between
    them (calls on one stream follow each other).  A call that is being captured
    gets its own, cleared inside the graph: the graph may be replayed on any
    stream."""
    if torch.cuda.is_current_stream_capturing():
        return torch.zeros(nbytes, dtype=torch.uint8, device=device)
    key = (device, stream)
    t = _WORKSPACES.get(key)
    if t is None or t.numel() < nbytes:
        t = _WORKSPACES[key] = torch.zeros(max(nbytes, 1 << 16), dtype=torch.uint8, device=device)
    return t


def _fail(kind, what, text):
    raise kind(f"{what}: {text}")


def _heads(what, name, t, dtype, device):
    """A [n, heads, dim] tensor of the call's type on the call's device."""
    if t.dim() != 3:
        _fail(ValueError, what, f"{name} must be [tokens, heads, dim], got {tuple(t.shape)}")
    if t.dtype != dtype or t.device != device:
        _fail(ValueError, what, f"{name} must be {dtype} on {device}, got {t.dtype} on {t.device}")
    if t.stride(2) != 1:
        _fail(NotImplementedError, what, f"{name}'s head vectors must be contiguous")
    if t.requires_grad and torch.is_grad_enabled():
        _fail(RuntimeError, what, f"{name} requires a gradient, which this operator does not have")


def _cache(what, name, t, like):
    if t.dim() != 4:
        _fail(ValueError, what, f"{name} must be [pages, page_size, kv_heads, dim], got {tuple(t.shape)}")
    if t.dtype != like.dtype or t.device != like.device:
        _fail(ValueError, what, f"{name} must be {like.dtype} on {like.device}, got {t.dtype} on {t.device}")
    if t.stride(3) != 1:
        _fail(NotImplementedError, what, f"{name}'s head vectors must be contiguous")


def _index(what, name, t, shape, device):
    if t.dtype != torch.int32 or t.device != device or tuple(t.shape) != shape:
        _fail(ValueError, what, f"{name} must be int32 {list(shape)} on {device}, got {t.dtype} "
                                f"{list(t.shape)} on {t.device}")
    if t.dim() and t.stride(-1) != 1 and t.shape[-1] > 1:
        _fail(NotImplementedError, what, f"{name} must be contiguous along its last axis")


def _kind(what, t):
    if t.device.type != "cuda":
        _fail(ValueError, what, f"needs CUDA tensors, got one on {t.device}")
    dt = _DTYPES.get(t.dtype)
    if dt is None:
        _fail(NotImplementedError, what, f"needs float16 or bfloat16, got {t.dtype}")
    return dt


def _call(fn, what, desc, device):
    if device.index != torch.cuda.current_device():
        with torch.cuda.device(device):
            rc = fn(C.byref(desc), torch.cuda.current_stream(device).cuda_stream)
    else:
        rc = fn(C.byref(desc), torch.cuda.current_stream(device).cuda_stream)
    if rc:
        msg = R.load_library().ktir_last_error().decode()
        raise (NotImplementedError if rc == -3 else ValueError if rc == -1 else RuntimeError)(msg or what)


def rotary_table(max_positions, rot, base=10000.0, device="cuda"):
    """The f32 table [max_positions, rot] of ``kv_append``: row p holds cos(p f_i),
    then sin(p f_i), f_i = base^(-2i/rot) for i < rot/2, formed in 64 bits."""
    if rot < 2 or rot % 2 or max_positions < 1:
        raise ValueError("rotary_table: needs an even rot and at least one position")
    i = torch.arange(rot // 2, dtype=torch.float64, device=device)
    angle = torch.arange(max_positions, dtype=torch.float64, device=device)[:, None] * float(base) ** (-2 * i / rot)
    return torch.cat([angle.cos(), angle.sin()], 1).float()


def kv_append(k, v, k_cache, v_cache, slots, q=None, positions=None, table=None, interleaved=False,
              q_out=None):
    """Write the keys and values of new tokens to their slots of a paged cache.

    k, v [tokens, kv_heads, dim]; slots [tokens] int32, slot s being place s %
    page_size of page s // page_size (negative: padding, not written); the slots
    of one call are distinct.  With `table` ([positions, rot] f32, see
    ``rotary_table``) and `positions` [tokens] int32, the first rot elements of
    every key are rotated by their position, in pairs (i, i + rot/2) or, when
    `interleaved`, (2i, 2i+1).  q [tokens, heads, dim], when given, is rotated
    likewise and returned (into `q_out`, which may be q itself)."""
    what = "kv_append"
    dt = _kind(what, k)
    device = k.device
    _heads(what, "k", k, k.dtype, device)
    _heads(what, "v", v, k.dtype, device)
    _cache(what, "k_cache", k_cache, k)
    _cache(what, "v_cache", v_cache, k)
    tokens, kv_heads, dim = k.shape
    if v.shape != k.shape:
        _fail(ValueError, what, f"v must have k's shape {tuple(k.shape)}, got {tuple(v.shape)}")
    if k_cache.shape != v_cache.shape or k_cache.shape[2] != kv_heads or k_cache.shape[3] != dim:
        _fail(ValueError, what, f"caches must be [pages, page_size, {kv_heads}, {dim}], got "
                                f"{tuple(k_cache.shape)} and {tuple(v_cache.shape)}")
    _index(what, "slots", slots, (tokens,), device)
    d = R.KtirKvAppendDesc()
    if table is not None:
        if positions is None:
            _fail(ValueError, what, "a table needs positions")
        _index(what, "positions", positions, (tokens,), device)
        if table.dim() != 2 or table.dtype != torch.float32 or table.device != device or table.stride(1) != 1:
            _fail(ValueError, what, f"table must be f32 [positions, rot] on {device}, rows contiguous")
        d.positions, d.table = positions.data_ptr(), table.data_ptr()
        d.table_rows, d.rot = table.shape
        d.table_stride = table.stride(0)
    elif positions is not None:
        _fail(ValueError, what, "positions need a table")
    heads = kv_heads
    if q is not None:
        _heads(what, "q", q, k.dtype, device)
        heads = q.shape[1]
        if q.shape[0] != tokens or q.shape[2] != dim:
            _fail(ValueError, what, f"q must be [{tokens}, heads, {dim}], got {tuple(q.shape)}")
        if q_out is None:
            q_out = torch.empty(q.shape, dtype=q.dtype, device=device)
        else:
            _heads(what, "q_out", q_out, k.dtype, device)
            if q_out.shape != q.shape:
                _fail(ValueError, what, f"q_out must have q's shape {tuple(q.shape)}, got {tuple(q_out.shape)}")
        d.q, d.q_out = q.data_ptr(), q_out.data_ptr()
        d.q_stride[0], d.q_stride[1], _ = q.stride()
        d.qo_stride[0], d.qo_stride[1], _ = q_out.stride()
    elif q_out is not None:
        _fail(ValueError, what, "q_out needs q")
    if tokens == 0 or kv_heads == 0 or heads == 0:
        return q_out
    d.k, d.v, d.k_cache, d.v_cache = k.data_ptr(), v.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr()
    d.slots, d.status = slots.data_ptr(), _status(device).data_ptr()
    d.tokens = tokens
    d.k_stride[0], d.k_stride[1], _ = k.stride()
    d.v_stride[0], d.v_stride[1], _ = v.stride()
    d.kc_stride[0], d.kc_stride[1], d.kc_stride[2], _ = k_cache.stride()
    d.vc_stride[0], d.vc_stride[1], d.vc_stride[2], _ = v_cache.stride()
    d.num_pages, d.page_size = k_cache.shape[0], k_cache.shape[1]
    d.heads, d.kv_heads, d.dim = heads, kv_heads, dim
    d.interleaved, d.dtype = 1 if interleaved else 0, dt
    _call(R.load_library().ktir_kv_append, what, d, device)
    return q_out


def _outputs(what, q, out, return_lse):
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    else:
        _heads(what, "out", out, q.dtype, q.device)
        if out.shape != q.shape:
            _fail(ValueError, what, f"out must have q's shape {tuple(q.shape)}, got {tuple(out.shape)}")
    lse = torch.empty(q.shape[:2], dtype=torch.float32, device=q.device) if return_lse else None
    return out, lse


def paged_decode(q, k_cache, v_cache, pages, lengths, scale=None, out=None, return_lse=False):
    """Attention of one new token per sequence over its cached keys and values.

    q [batch, heads, dim]; pages [batch, max_pages] int32, a sequence's pages in
    order (entries past its length are not read); lengths [batch] int32, the keys
    of each sequence, the new token's own included (append it first).  heads is
    a multiple of the caches' kv_heads: head h reads kv head h // (heads //
    kv_heads).  scale defaults to dim ** -0.5.  Returns out [batch, heads, dim],
    zero where a length is 0; with `return_lse` also the f32 [batch, heads]
    logarithm of each row's sum of exponentials (-inf for length 0)."""
    what = "paged_decode"
    dt = _kind(what, q)
    device = q.device
    _heads(what, "q", q, q.dtype, device)
    _cache(what, "k_cache", k_cache, q)
    _cache(what, "v_cache", v_cache, q)
    batch, heads, dim = q.shape
    num_pages, page_size, kv_heads, _ = k_cache.shape
    if k_cache.shape != v_cache.shape or k_cache.shape[3] != dim or not kv_heads or heads % kv_heads:
        _fail(ValueError, what, f"caches must be [pages, page_size, kv_heads, {dim}] with kv_heads dividing "
                                f"{heads}, got {tuple(k_cache.shape)} and {tuple(v_cache.shape)}")
    if pages.dim() != 2:
        _fail(ValueError, what, f"pages must be [batch, max_pages], got {tuple(pages.shape)}")
    _index(what, "pages", pages, (batch, pages.shape[1]), device)
    _index(what, "lengths", lengths, (batch,), device)
    out, lse = _outputs(what, q, out, return_lse)
    if batch and heads:
        lib = R.load_library()
        d = R.KtirPagedDecodeDesc()
        need = lib.ktir_paged_decode_workspace(batch, heads, kv_heads, dim)
        ws = _workspace(need, device, torch.cuda.current_stream(device).cuda_stream)
        d.q, d.k_cache, d.v_cache, d.out = q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), out.data_ptr()
        if lse is not None:
            d.lse = lse.data_ptr()
        d.pages, d.lengths = pages.data_ptr(), lengths.data_ptr()
        d.workspace, d.workspace_bytes = ws.data_ptr(), ws.numel()
        d.status = _status(device).data_ptr()
        d.batch, d.max_pages, d.page_row = batch, pages.shape[1], pages.stride(0)
        d.num_pages, d.page_size = num_pages, page_size
        d.q_stride[0], d.q_stride[1], _ = q.stride()
        d.out_stride[0], d.out_stride[1], _ = out.stride()
        d.kc_stride[0], d.kc_stride[1], d.kc_stride[2], _ = k_cache.stride()
        d.vc_stride[0], d.vc_stride[1], d.vc_stride[2], _ = v_cache.stride()
        d.heads, d.kv_heads, d.dim, d.dtype = heads, kv_heads, dim, dt
        d.scale = dim ** -0.5 if scale is None else scale
        _call(lib.ktir_paged_decode, what, d, device)
    return (out, lse) if return_lse else out


def prompt_attention(q, k, v, offsets, kv_offsets=None, causal=True, scale=None, out=None,
                     return_lse=False):
    """Attention over packed prompts of different lengths.

    q [tokens, heads, dim], k and v [kv_tokens, kv_heads, dim]; sequence b's
    queries are tokens offsets[b] .. offsets[b + 1] - 1 (offsets [batch + 1]
    int32, from 0 to tokens), its keys tokens kv_offsets[b] .. kv_offsets[b + 1]
    - 1 (default: offsets).  A causal mask is aligned at the end: query i of n
    sees keys j <= i + m - n of m, so later pieces of a prompt attend to its
    earlier ones.  heads is a multiple of kv_heads, scale defaults to dim **
    -0.5.  Returns out [tokens, heads, dim], zero where a query sees no key; with
    `return_lse` also the f32 [tokens, heads] logarithm of each row's sum of
    exponentials."""
    what = "prompt_attention"
    dt = _kind(what, q)
    device = q.device
    _heads(what, "q", q, q.dtype, device)
    _heads(what, "k", k, q.dtype, device)
    _heads(what, "v", v, q.dtype, device)
    tokens, heads, dim = q.shape
    kv_tokens, kv_heads, _ = k.shape
    if k.shape != v.shape or k.shape[2] != dim or not kv_heads or heads % kv_heads:
        _fail(ValueError, what, f"k and v must be [kv_tokens, kv_heads, {dim}] with kv_heads dividing {heads}, "
                                f"got {tuple(k.shape)} and {tuple(v.shape)}")
    if offsets.dim() != 1 or offsets.shape[0] < 2:
        _fail(ValueError, what, f"offsets must be [batch + 1], got {tuple(offsets.shape)}")
    _index(what, "offsets", offsets, tuple(offsets.shape), device)
    if kv_offsets is None:
        kv_offsets = offsets
        if kv_tokens != tokens:
            _fail(ValueError, what, f"{tokens} queries and {kv_tokens} keys need kv_offsets")
    else:
        _index(what, "kv_offsets", kv_offsets, tuple(offsets.shape), device)
    out, lse = _outputs(what, q, out, return_lse)
    if tokens and heads:
        lib = R.load_library()
        d = R.KtirPromptDesc()
        d.q, d.k, d.v, d.out = q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr()
        if lse is not None:
            d.lse = lse.data_ptr()
        d.offsets, d.kv_offsets = offsets.data_ptr(), kv_offsets.data_ptr()
        d.status = _status(device).data_ptr()
        d.batch, d.tokens, d.kv_tokens = offsets.shape[0] - 1, tokens, kv_tokens
        d.q_stride[0], d.q_stride[1], _ = q.stride()
        d.k_stride[0], d.k_stride[1], _ = k.stride()
        d.v_stride[0], d.v_stride[1], _ = v.stride()
        d.out_stride[0], d.out_stride[1], _ = out.stride()
        d.heads, d.kv_heads, d.dim, d.dtype = heads, kv_heads, dim, dt
        d.scale = dim ** -0.5 if scale is None else scale
        d.causal = 1 if causal else 0
        _call(lib.ktir_prompt_attention, what, d, device)
    return (out, lse) if return_lse else out
