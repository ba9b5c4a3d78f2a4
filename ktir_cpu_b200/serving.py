"""Serving operators of a decoder: a paged key-value cache and the attention on it.

    kv_append         rotate new keys (and queries) by their positions, write
                      keys and values to their slots of a paged cache
    prompt_attention  (causal) attention over packed prompts, grouped heads
    paged_decode      attention of one new token per sequence over its cache

They work on torch CUDA tensors (f16 or bf16, sums in f32), run on the current
stream of the tensors' device, allocate nothing but their outputs and a
workspace per stream (and per stream of a capture), wait for nothing and can be
captured into a CUDA graph.
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

import importlib

import torch

from . import runtime as R

_DTYPES = (torch.float16, torch.bfloat16)
_EXT = None


def _ext():
    """The compiled binding (never falls back to anything else)."""
    global _EXT
    if _EXT is None:
        R.load_library()
        try:
            _EXT = importlib.import_module("._serving", __package__)
        except ImportError as e:
            raise RuntimeError(f"{R.binding_path()} is missing or does not load: build it with "
                               "`python -m ktir_cpu_b200.build`") from e
    return _EXT


def check_status(device=None) -> None:
    """Wait for `device` (default: the current one) and raise for what the
    serving operators have reported there since the last check: RuntimeError if a
    wait inside a kernel ran out (some of the outputs since then were given up),
    else IndexError for an index out of range."""
    dev = torch.cuda.current_device() if device is None else torch.device(device).index
    if dev is None:
        dev = torch.cuda.current_device()
    t = _ext().status(dev)
    if t is None:
        return
    torch.cuda.synchronize(dev)
    v = int(t.item())
    if v:
        t.zero_()
        torch.cuda.synchronize(dev)
    index = "a page, slot, position, length or offset of a serving operator is out of range"
    if v & R.STATUS_TIMEOUT:             # the graver one: an IndexError alone would let the outputs pass
        _ext().forget(dev)               # the call that was given up may have left counters part-counted
        raise RuntimeError("device wait timed out" + (f"; and {index}" if v & R.STATUS_BAD_INDEX else ""))
    if v & R.STATUS_BAD_INDEX:
        raise IndexError(index)


# -- what is wrong with a call that did not pass its operator's check ----------------
def _fail(kind, what, text):
    raise kind(f"{what}: {text}")


def _tensor(what, name, t):
    if not isinstance(t, torch.Tensor):
        _fail(ValueError, what, f"{name} must be a tensor, got {type(t).__name__}")


def _kind(what, name, t):
    _tensor(what, name, t)
    if t.device.type != "cuda":
        _fail(ValueError, what, f"needs CUDA tensors, got one on {t.device}")
    if t.dtype not in _DTYPES:
        _fail(NotImplementedError, what, f"needs float16 or bfloat16, got {t.dtype}")


def _no_gradient(what, name, t):
    if t.requires_grad and torch.is_grad_enabled():
        _fail(RuntimeError, what, f"{name} requires a gradient, which this operator does not have")
    if torch._C._is_fwd_grad_enabled() and torch.autograd.forward_ad.unpack_dual(t).tangent is not None:
        _fail(RuntimeError, what, f"{name} has a forward-mode tangent, which this operator does not carry on")


def _vectors(what, name, t, like, layout):
    """A tensor of head vectors, of the call's type and device."""
    _tensor(what, name, t)
    if t.dim() != layout.count(",") + 1:
        _fail(ValueError, what, f"{name} must be {layout}, got {tuple(t.shape)}")
    if t.dtype != like.dtype or t.device != like.device:
        _fail(ValueError, what, f"{name} must be {like.dtype} on {like.device}, got {t.dtype} on {t.device}")
    if t.stride(-1) != 1:
        _fail(NotImplementedError, what, f"{name}'s head vectors must be contiguous")
    _no_gradient(what, name, t)


def _heads(what, name, t, like):
    _vectors(what, name, t, like, "[tokens, heads, dim]")


def _cache(what, name, t, like):
    _vectors(what, name, t, like, "[pages, page_size, kv_heads, dim]")


def _index(what, name, t, shape, like):
    _tensor(what, name, t)
    if t.dtype != torch.int32 or t.device != like.device or tuple(t.shape) != tuple(shape):
        _fail(ValueError, what, f"{name} must be int32 {list(shape)} on {like.device}, got {t.dtype} "
                                f"{list(t.shape)} on {t.device}")
    if t.dim() and t.stride(-1) != 1 and t.shape[-1] > 1:
        _fail(NotImplementedError, what, f"{name} must be contiguous along its last axis")


def _same_shape(what, name, t, other, of):
    if t.shape != other.shape:
        _fail(ValueError, what, f"{name} must have {of}'s shape {tuple(other.shape)}, got {tuple(t.shape)}")


def _out(what, out, q):
    if out is not None:
        _heads(what, "out", out, q)
        _same_shape(what, "out", out, q, "q")


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
    _kind(what, "k", k)
    _heads(what, "k", k, k)
    _heads(what, "v", v, k)
    _cache(what, "k_cache", k_cache, k)
    _cache(what, "v_cache", v_cache, k)
    _same_shape(what, "v", v, k, "k")
    tokens, kv_heads, dim = k.shape
    if not kv_heads:
        _fail(ValueError, what, "k and v have no heads")
    if k_cache.shape != v_cache.shape or tuple(k_cache.shape[2:]) != (kv_heads, dim):
        _fail(ValueError, what, f"caches must be [pages, page_size, {kv_heads}, {dim}], got "
                                f"{tuple(k_cache.shape)} and {tuple(v_cache.shape)}")
    _index(what, "slots", slots, (tokens,), k)
    if (positions is None) != (table is None):
        _fail(ValueError, what, "positions and table go together")
    if table is not None:
        _tensor(what, "table", table)
        _index(what, "positions", positions, (tokens,), k)
        if table.dim() != 2 or table.dtype != torch.float32 or table.device != k.device or table.stride(1) != 1:
            _fail(ValueError, what, f"table must be f32 [positions, rot] on {k.device}, rows contiguous")
        _no_gradient(what, "table", table)
    if q is not None:
        _heads(what, "q", q, k)
        if q.shape[0] != tokens or q.shape[2] != dim:
            _fail(ValueError, what, f"q must be [{tokens}, heads, {dim}], got {tuple(q.shape)}")
    elif q_out is not None:
        _fail(ValueError, what, "q_out needs q")
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
    likewise and returned (into `q_out`, which may be q itself).  A token whose slot
    is past the cache is not written to it; one whose position is not in the table
    isn't either, and its query comes back as zeros (both reported by
    ``check_status``; the position of padding is not)."""
    r = _ext().kv_append(k, v, k_cache, v_cache, slots, q, positions, table, interleaved, q_out)
    if r is NotImplemented:
        _wrong_append(k, v, k_cache, v_cache, slots, q, positions, table, q_out)
    return r


def _wrong_decode(q, k_cache, v_cache, pages, lengths, out):
    what = "paged_decode"
    _kind(what, "q", q)
    _heads(what, "q", q, q)
    _cache(what, "k_cache", k_cache, q)
    _cache(what, "v_cache", v_cache, q)
    batch, heads, dim = q.shape
    kv_heads = k_cache.shape[2]
    if k_cache.shape != v_cache.shape or k_cache.shape[3] != dim or not kv_heads or heads % kv_heads:
        _fail(ValueError, what, f"caches must be [pages, page_size, kv_heads, {dim}] with kv_heads dividing "
                                f"{heads}, got {tuple(k_cache.shape)} and {tuple(v_cache.shape)}")
    _tensor(what, "pages", pages)
    if pages.dim() != 2:
        _fail(ValueError, what, f"pages must be [batch, max_pages], got {tuple(pages.shape)}")
    _index(what, "pages", pages, (batch, pages.shape[1]), q)
    _index(what, "lengths", lengths, (batch,), q)
    _out(what, out, q)
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
    r = _ext().paged_decode(q, k_cache, v_cache, pages, lengths, scale, out, return_lse)
    if r is NotImplemented:
        _wrong_decode(q, k_cache, v_cache, pages, lengths, out)
    return r


def _wrong_prompt(q, k, v, offsets, kv_offsets, out):
    what = "prompt_attention"
    _kind(what, "q", q)
    _heads(what, "q", q, q)
    _heads(what, "k", k, q)
    _heads(what, "v", v, q)
    tokens, heads, dim = q.shape
    kv_heads = k.shape[1]
    if k.shape != v.shape or k.shape[2] != dim or not kv_heads or heads % kv_heads:
        _fail(ValueError, what, f"k and v must be [kv_tokens, kv_heads, {dim}] with kv_heads dividing {heads}, "
                                f"got {tuple(k.shape)} and {tuple(v.shape)}")
    _tensor(what, "offsets", offsets)
    if offsets.dim() != 1 or offsets.shape[0] < 2:
        _fail(ValueError, what, f"offsets must be [batch + 1], got {tuple(offsets.shape)}")
    _index(what, "offsets", offsets, tuple(offsets.shape), q)
    if kv_offsets is not None:
        _index(what, "kv_offsets", kv_offsets, tuple(offsets.shape), q)
    elif tokens != k.shape[0]:
        _fail(ValueError, what, f"{tokens} queries and {k.shape[0]} keys need kv_offsets")
    _out(what, out, q)
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
    -0.5.  A value row that is not finite reaches, besides the queries that see it,
    some just before it, as 0 times it is not 0 in the product: the mask leaves out
    whole blocks of keys only, 80 of them at dim 128 and 128 at dim 64, for tiles of
    128 // (heads // kv_heads) tokens, so that queries less than the sum of the two
    before it may be reached.  A key row does not, nor does either reach another
    sequence.
    Returns out [tokens, heads, dim], zero where a query sees no key (and, if
    offsets are bad, where it belongs to no sequence); with `return_lse` also the f32 [tokens, heads] logarithm of each row's sum of
    exponentials."""
    r = _ext().prompt_attention(q, k, v, offsets, kv_offsets, causal, scale, out, return_lse)
    if r is NotImplemented:
        _wrong_prompt(q, k, v, offsets, kv_offsets, out)
    return r
