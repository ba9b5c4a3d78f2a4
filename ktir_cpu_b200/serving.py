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

import struct

import torch

from . import runtime as R

_DTYPES = {torch.float16: R.F16, torch.bfloat16: R.BF16}
_I32 = torch.int32
_STATUS = {}
_WORKSPACES = {}
_LIB = None

# The descriptors of include/ktir_b200.h, packed in one go: a call of few tokens
# takes the GPU a few microseconds, about what setting the fields one by one costs.
_APPEND = struct.Struct("10Q q 2q2q2q2q 3q3q 2q 2q 4i 2i")
_DECODE = struct.Struct("9Q q 3q 2q 2q2q 3q3q 4i f i")
_PROMPT = struct.Struct("8Q 3q 2q2q2q2q 4i f i")


def _lib():
    global _LIB
    if _LIB is None:
        _LIB = R.load_library()
    return _LIB


def _status(dev):
    t = _STATUS.get(dev)
    if t is None:
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("call a serving operator once on this device before capturing it")
        t = _STATUS[dev] = torch.zeros(1, dtype=_I32, device=torch.device("cuda", dev))
        torch.cuda.synchronize(dev)   # whichever stream uses it next finds it cleared
    return t.data_ptr()


def check_status(device=None) -> None:
    """Wait for `device` (default: the current one) and raise for what the
    serving operators have reported there since the last check."""
    dev = torch.cuda.current_device() if device is None else torch.device(device).index
    if dev is None:
        dev = torch.cuda.current_device()
    t = _STATUS.get(dev)
    if t is None:
        return
    torch.cuda.synchronize(dev)
    v = int(t.item())
    if v:
        t.zero_()
        torch.cuda.synchronize(dev)
    if v & R.STATUS_BAD_INDEX:
        raise IndexError("a page, slot, position, length or offset of a serving operator is out of range")
    if v & R.STATUS_TIMEOUT:
        raise RuntimeError("device wait timed out")


def _stream(dev):
    return torch.cuda.current_stream(dev).cuda_stream


# the stream's handle alone, where this torch offers it (a tenth of the time)
_stream = getattr(torch._C, "_cuda_getCurrentRawStream", _stream)


def _workspace(nbytes, dev, stream):
    """Zeroed scratch of at least `nbytes` for calls on `stream`, kept between
    them (calls on one stream follow each other).  A call that is being captured
    gets its own, cleared inside the graph: the graph may be replayed on any
    stream."""
    if torch.cuda.is_current_stream_capturing():
        return torch.zeros(nbytes, dtype=torch.uint8, device=torch.device("cuda", dev))
    key = (dev, stream)
    t = _WORKSPACES.get(key)
    if t is None or t.numel() < nbytes:
        t = _WORKSPACES[key] = torch.zeros(nbytes + (nbytes >> 2), dtype=torch.uint8,
                                           device=torch.device("cuda", dev))
    return t


def _run(fn, what, desc, dev, stream):
    """One C call; `desc` are the descriptor's bytes."""
    if dev != torch.cuda.current_device():
        with torch.cuda.device(dev):
            rc = fn(desc, stream)
    else:
        rc = fn(desc, stream)
    if rc:
        msg = _lib().ktir_last_error().decode()
        raise (NotImplementedError if rc == -3 else ValueError if rc == -1 else RuntimeError)(msg or what)


# -- what is wrong with a call that did not pass its operator's check ----------------
def _fail(kind, what, text):
    raise kind(f"{what}: {text}")


def _kind(what, t):
    if t.device.type != "cuda":
        _fail(ValueError, what, f"needs CUDA tensors, got one on {t.device}")
    if t.dtype not in _DTYPES:
        _fail(NotImplementedError, what, f"needs float16 or bfloat16, got {t.dtype}")


def _vectors(what, name, t, like, layout):
    """A tensor of head vectors, of the call's type and device."""
    if t.dim() != layout.count(",") + 1:
        _fail(ValueError, what, f"{name} must be {layout}, got {tuple(t.shape)}")
    if t.dtype != like.dtype or t.device != like.device:
        _fail(ValueError, what, f"{name} must be {like.dtype} on {like.device}, got {t.dtype} on {t.device}")
    if t.stride(-1) != 1:
        _fail(NotImplementedError, what, f"{name}'s head vectors must be contiguous")
    if t.requires_grad and torch.is_grad_enabled():
        _fail(RuntimeError, what, f"{name} requires a gradient, which this operator does not have")


def _heads(what, name, t, like):
    _vectors(what, name, t, like, "[tokens, heads, dim]")


def _cache(what, name, t, like):
    _vectors(what, name, t, like, "[pages, page_size, kv_heads, dim]")


def _index(what, name, t, shape, like):
    if t.dtype != _I32 or t.device != like.device or tuple(t.shape) != tuple(shape):
        _fail(ValueError, what, f"{name} must be int32 {list(shape)} on {like.device}, got {t.dtype} "
                                f"{list(t.shape)} on {t.device}")
    if t.dim() and t.stride(-1) != 1 and t.shape[-1] > 1:
        _fail(NotImplementedError, what, f"{name} must be contiguous along its last axis")


def _same_shape(what, name, t, other, of):
    if t.shape != other.shape:
        _fail(ValueError, what, f"{name} must have {of}'s shape {tuple(other.shape)}, got {tuple(t.shape)}")


def _unwanted_grad(*ts):
    return torch.is_grad_enabled() and any(t.requires_grad for t in ts)


def rotary_table(max_positions, rot, base=10000.0, device="cuda"):
    """The f32 table [max_positions, rot] of ``kv_append``: row p holds cos(p f_i),
    then sin(p f_i), f_i = base^(-2i/rot) for i < rot/2, formed in 64 bits."""
    if rot < 2 or rot % 2 or max_positions < 1:
        raise ValueError("rotary_table: needs an even rot and at least one position")
    i = torch.arange(rot // 2, dtype=torch.float64, device=device)
    angle = torch.arange(max_positions, dtype=torch.float64, device=device)[:, None] * float(base) ** (-2 * i / rot)
    return torch.cat([angle.cos(), angle.sin()], 1).float()


def _wrong_append(k, v, k_cache, v_cache, slots, q, positions, table, q_out):
    what = "kv_append"
    _kind(what, k)
    _heads(what, "k", k, k)
    _heads(what, "v", v, k)
    _cache(what, "k_cache", k_cache, k)
    _cache(what, "v_cache", v_cache, k)
    _same_shape(what, "v", v, k, "k")
    tokens, kv_heads, dim = k.shape
    if k_cache.shape != v_cache.shape or tuple(k_cache.shape[2:]) != (kv_heads, dim):
        _fail(ValueError, what, f"caches must be [pages, page_size, {kv_heads}, {dim}], got "
                                f"{tuple(k_cache.shape)} and {tuple(v_cache.shape)}")
    _index(what, "slots", slots, (tokens,), k)
    if (positions is None) != (table is None):
        _fail(ValueError, what, "positions and table go together")
    if table is not None:
        _index(what, "positions", positions, (tokens,), k)
        if table.dim() != 2 or table.dtype != torch.float32 or table.device != k.device or table.stride(1) != 1:
            _fail(ValueError, what, f"table must be f32 [positions, rot] on {k.device}, rows contiguous")
    if q is None:
        _fail(ValueError, what, "q_out needs q")
    _heads(what, "q", q, k)
    if q.shape[0] != tokens or q.shape[2] != dim:
        _fail(ValueError, what, f"q must be [{tokens}, heads, {dim}], got {tuple(q.shape)}")
    if q_out is not None:
        _heads(what, "q_out", q_out, k)
        _same_shape(what, "q_out", q_out, q, "q")
    _fail(ValueError, what, "arguments that do not fit together")


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
    dt, dev, typ = _DTYPES.get(k.dtype), k.get_device(), k.dtype
    ks, cs = k.shape, k_cache.shape
    k_st, v_st, kc_st, vc_st = k.stride(), v.stride(), k_cache.stride(), v_cache.stride()
    if not (dt is not None and dev >= 0 and len(ks) == 3 and len(cs) == 4 and v.shape == ks
            and v_cache.shape == cs and cs[2] == ks[1] and cs[3] == ks[2]
            and v.dtype is typ and k_cache.dtype is typ and v_cache.dtype is typ and slots.dtype is _I32
            and v.get_device() == dev and k_cache.get_device() == dev and v_cache.get_device() == dev
            and slots.get_device() == dev and k_st[2] == 1 and v_st[2] == 1 and kc_st[3] == 1 and vc_st[3] == 1
            and slots.shape == ks[:1] and (slots.stride(0) == 1 or ks[0] <= 1)
            and not _unwanted_grad(k, v, k_cache, v_cache)):
        _wrong_append(k, v, k_cache, v_cache, slots, q, positions, table, q_out)
    tokens, heads, dim = ks
    kv_heads = heads
    q_at = out_at = at = rows = 0
    rot = row = q0 = q1 = o0 = o1 = 0
    if table is not None or positions is not None:
        if not (table is not None and positions is not None and positions.dtype is _I32
                and positions.get_device() == dev and positions.shape == ks[:1]
                and (positions.stride(0) == 1 or tokens <= 1) and table.dtype is torch.float32
                and table.get_device() == dev and table.dim() == 2 and table.stride(1) == 1):
            _wrong_append(k, v, k_cache, v_cache, slots, q, positions, table, q_out)
        at, rows = positions.data_ptr(), table.data_ptr()
        row, rot = table.stride(0), table.shape[1]
    if q is not None or q_out is not None:
        if q is not None and q_out is None:
            q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
        if not (q is not None and q.dim() == 3 and q.shape[0] == tokens and q.shape[2] == dim
                and q_out.shape == q.shape and q.dtype is typ and q_out.dtype is typ
                and q.get_device() == dev and q_out.get_device() == dev and q.stride(2) == 1
                and q_out.stride(2) == 1 and not _unwanted_grad(q, q_out)):
            _wrong_append(k, v, k_cache, v_cache, slots, q, positions, table, q_out)
        heads = q.shape[1]
        q_at, out_at = q.data_ptr(), q_out.data_ptr()
        (q0, q1, _), (o0, o1, _) = q.stride(), q_out.stride()
    if tokens == 0 or kv_heads == 0 or heads == 0:
        return q_out
    desc = _APPEND.pack(
        q_at, k.data_ptr(), v.data_ptr(), out_at, k_cache.data_ptr(), v_cache.data_ptr(), slots.data_ptr(),
        at, rows, _status(dev), tokens, q0, q1, k_st[0], k_st[1], v_st[0], v_st[1], o0, o1,
        kc_st[0], kc_st[1], kc_st[2], vc_st[0], vc_st[1], vc_st[2], cs[0], cs[1],
        table.shape[0] if rows else 0, row, heads, kv_heads, dim, rot, 1 if interleaved else 0, dt)
    _run(_lib().ktir_kv_append, "kv_append", desc, dev, _stream(dev))
    return q_out


def _outputs(what, q, out, return_lse):
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    else:
        _heads(what, "out", out, q)
        _same_shape(what, "out", out, q, "q")
    lse = torch.empty(q.shape[:2], dtype=torch.float32, device=q.device) if return_lse else None
    return out, lse


def _wrong_decode(q, k_cache, v_cache, pages, lengths):
    what = "paged_decode"
    _kind(what, q)
    _heads(what, "q", q, q)
    _cache(what, "k_cache", k_cache, q)
    _cache(what, "v_cache", v_cache, q)
    batch, heads, dim = q.shape
    kv_heads = k_cache.shape[2]
    if k_cache.shape != v_cache.shape or k_cache.shape[3] != dim or not kv_heads or heads % kv_heads:
        _fail(ValueError, what, f"caches must be [pages, page_size, kv_heads, {dim}] with kv_heads dividing "
                                f"{heads}, got {tuple(k_cache.shape)} and {tuple(v_cache.shape)}")
    if pages.dim() != 2:
        _fail(ValueError, what, f"pages must be [batch, max_pages], got {tuple(pages.shape)}")
    _index(what, "pages", pages, (batch, pages.shape[1]), q)
    _index(what, "lengths", lengths, (batch,), q)
    _fail(ValueError, what, "arguments that do not fit together")


def paged_decode(q, k_cache, v_cache, pages, lengths, scale=None, out=None, return_lse=False):
    """Attention of one new token per sequence over its cached keys and values.

    q [batch, heads, dim]; pages [batch, max_pages] int32, a sequence's pages in
    order (entries past its length are not read); lengths [batch] int32, the keys
    of each sequence, the new token's own included (append it first).  heads is
    a multiple of the caches' kv_heads: head h reads kv head h // (heads //
    kv_heads).  scale defaults to dim ** -0.5.  Returns out [batch, heads, dim],
    zero where a length is 0; with `return_lse` also the f32 [batch, heads]
    logarithm of each row's sum of exponentials (-inf for length 0)."""
    dt, dev, typ = _DTYPES.get(q.dtype), q.get_device(), q.dtype
    qs, cs, ps = q.shape, k_cache.shape, pages.shape
    q_st, kc_st, vc_st, p_st = q.stride(), k_cache.stride(), v_cache.stride(), pages.stride()
    if not (dt is not None and dev >= 0 and len(qs) == 3 and len(cs) == 4 and len(ps) == 2
            and v_cache.shape == cs and cs[3] == qs[2] and cs[2] and qs[1] % cs[2] == 0 and ps[0] == qs[0]
            and lengths.shape == qs[:1] and k_cache.dtype is typ and v_cache.dtype is typ
            and pages.dtype is _I32 and lengths.dtype is _I32 and k_cache.get_device() == dev
            and v_cache.get_device() == dev and pages.get_device() == dev and lengths.get_device() == dev
            and q_st[2] == 1 and kc_st[3] == 1 and vc_st[3] == 1 and (p_st[1] == 1 or ps[1] <= 1)
            and (lengths.stride(0) == 1 or qs[0] <= 1) and not _unwanted_grad(q, k_cache, v_cache)):
        _wrong_decode(q, k_cache, v_cache, pages, lengths)
    out, lse = _outputs("paged_decode", q, out, return_lse)
    batch, heads, dim = qs
    if batch and heads:
        lib, stream = _lib(), _stream(dev)
        ws = _workspace(lib.ktir_paged_decode_workspace(batch, heads, cs[2], dim), dev, stream)
        o_st = out.stride()
        desc = _DECODE.pack(
            q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), out.data_ptr(),
            lse.data_ptr() if return_lse else 0, pages.data_ptr(), lengths.data_ptr(), ws.data_ptr(),
            _status(dev), ws.numel(), batch, ps[1], p_st[0], cs[0], cs[1], q_st[0], q_st[1], o_st[0], o_st[1],
            kc_st[0], kc_st[1], kc_st[2], vc_st[0], vc_st[1], vc_st[2], heads, cs[2], dim, dt,
            dim ** -0.5 if scale is None else scale, 0)
        _run(lib.ktir_paged_decode, "paged_decode", desc, dev, stream)
    return (out, lse) if return_lse else out


def _wrong_prompt(q, k, v, offsets, kv_offsets):
    what = "prompt_attention"
    _kind(what, q)
    _heads(what, "q", q, q)
    _heads(what, "k", k, q)
    _heads(what, "v", v, q)
    tokens, heads, dim = q.shape
    kv_heads = k.shape[1]
    if k.shape != v.shape or k.shape[2] != dim or not kv_heads or heads % kv_heads:
        _fail(ValueError, what, f"k and v must be [kv_tokens, kv_heads, {dim}] with kv_heads dividing {heads}, "
                                f"got {tuple(k.shape)} and {tuple(v.shape)}")
    if offsets.dim() != 1 or offsets.shape[0] < 2:
        _fail(ValueError, what, f"offsets must be [batch + 1], got {tuple(offsets.shape)}")
    _index(what, "offsets", offsets, tuple(offsets.shape), q)
    if kv_offsets is None:
        _fail(ValueError, what, f"{tokens} queries and {k.shape[0]} keys need kv_offsets")
    _index(what, "kv_offsets", kv_offsets, tuple(offsets.shape), q)
    _fail(ValueError, what, "arguments that do not fit together")


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
    dt, dev, typ = _DTYPES.get(q.dtype), q.get_device(), q.dtype
    qs, ks, os = q.shape, k.shape, offsets.shape
    q_st, k_st, v_st = q.stride(), k.stride(), v.stride()
    if not (dt is not None and dev >= 0 and len(qs) == 3 and len(ks) == 3 and v.shape == ks and ks[2] == qs[2]
            and ks[1] and qs[1] % ks[1] == 0 and len(os) == 1 and os[0] >= 2 and k.dtype is typ
            and v.dtype is typ and offsets.dtype is _I32 and k.get_device() == dev and v.get_device() == dev
            and offsets.get_device() == dev and q_st[2] == 1 and k_st[2] == 1 and v_st[2] == 1
            and offsets.stride(0) == 1 and not _unwanted_grad(q, k, v)
            and (ks[0] == qs[0] if kv_offsets is None else
                 kv_offsets.dtype is _I32 and kv_offsets.shape == os and kv_offsets.get_device() == dev
                 and kv_offsets.stride(0) == 1)):
        _wrong_prompt(q, k, v, offsets, kv_offsets)
    out, lse = _outputs("prompt_attention", q, out, return_lse)
    tokens, heads, dim = qs
    if tokens and heads:
        o_st = out.stride()
        at = offsets.data_ptr()
        desc = _PROMPT.pack(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr() if return_lse else 0,
            at, at if kv_offsets is None else kv_offsets.data_ptr(), _status(dev), os[0] - 1, tokens, ks[0],
            q_st[0], q_st[1], k_st[0], k_st[1], v_st[0], v_st[1], o_st[0], o_st[1], heads, ks[1], dim, dt,
            dim ** -0.5 if scale is None else scale, 1 if causal else 0)
        _run(_lib().ktir_prompt_attention, "prompt_attention", desc, dev, _stream(dev))
    return (out, lse) if return_lse else out
