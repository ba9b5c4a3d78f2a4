"""The serving operators (paged append, packed prompts, single-token decode)
against plain 64-bit forms; bounds derived in serving_util.py."""

import math
import random

import pytest

import serving_util as S

pytestmark = pytest.mark.gpu


def _gen(seed):
    import torch
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(gen, typ, *shape):
    import torch
    return torch.randn(*shape, generator=gen, device="cuda").to(S.dtype_of(typ))


def _cache(gen, typ, pages, page, heads, dim, head_major):
    if head_major:
        return _randn(gen, typ, pages, heads, page, dim).transpose(1, 2)
    return _randn(gen, typ, pages, page, heads, dim)


# -- append -----------------------------------------------------------------------

@pytest.mark.parametrize("typ,tokens,heads,kv_heads,dim,rot,page,interleaved,head_major", [
    ("bf16", 1, 8, 2, 128, 128, 16, False, False),
    ("f16", 37, 4, 4, 64, 32, 8, True, True),
    ("bf16", 300, 6, 3, 96, 96, 24, False, True),
    ("f16", 65, 40, 8, 128, 64, 1, False, False),
    ("bf16", 9, 1, 1, 256, 16, 128, True, False),
    ("f16", 12, 3, 1, 80, 0, 7, False, False),
])
def test_append(typ, tokens, heads, kv_heads, dim, rot, page, interleaved, head_major):
    import torch
    from ktir_cpu_b200 import check_status, kv_append, rotary_table
    gen = _gen(tokens)
    pages = tokens // page + 3
    qkv = _randn(gen, typ, tokens, heads + 2 * kv_heads, dim)
    q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv_heads], qkv[:, heads + kv_heads:]
    kc, vc = (_cache(gen, typ, pages, page, kv_heads, dim, head_major) for _ in range(2))
    kc0, vc0 = kc.clone(), vc.clone()
    slots = torch.randperm(pages * page, generator=gen, device="cuda")[:tokens].int()
    if tokens > 1:
        slots[::7] = -1
    args = {}
    if rot:
        args = dict(table=rotary_table(5000, rot), interleaved=interleaved,
                    positions=torch.randint(0, 5000, (tokens,), generator=gen, device="cuda").int())
    q0 = qkv.clone()
    out = kv_append(k, v, kc, vc, slots, q=q, **args)
    check_status()
    assert torch.equal(qkv, q0), "inputs changed"
    def turned(x):
        return S.rotate(x, args["table"], args["positions"], interleaved) if rot else (x.double(), torch.zeros_like(x, dtype=torch.float64))
    want, bound = turned(q)
    assert ((out.double() - want).abs() <= bound).all()
    kept = slots >= 0
    at = (slots[kept].long() // page, slots[kept].long() % page)
    want, bound = turned(k)
    assert ((kc[at].double() - want[kept]).abs() <= bound[kept]).all()
    assert torch.equal(vc[at], v[kept])
    kc0[at], vc0[at] = kc[at], vc[at]
    assert torch.equal(kc, kc0) and torch.equal(vc, vc0), "another slot was written"


def test_append_in_place_and_without_queries():
    import torch
    from ktir_cpu_b200 import check_status, kv_append, rotary_table
    gen = _gen(3)
    k, v, q = (_randn(gen, "bf16", 20, 4, 64) for _ in range(3))
    caches = [torch.zeros(4, 8, 4, 64, dtype=torch.bfloat16, device="cuda") for _ in range(4)]
    slots = torch.arange(20, dtype=torch.int32, device="cuda")
    args = dict(positions=slots, table=rotary_table(64, 64))
    out = kv_append(k, v, caches[0], caches[1], slots, q=q, **args)
    same = q.clone()
    assert kv_append(k, v, caches[2], caches[3], slots, q=same, q_out=same, **args) is same
    assert torch.equal(out, same) and torch.equal(caches[0], caches[2]) and torch.equal(caches[1], caches[3])
    caches[2].zero_()
    assert kv_append(k, v, caches[2], caches[3], slots, **args) is None
    assert torch.equal(caches[0], caches[2])
    check_status()


def test_append_reports_bad_indices():
    import torch
    from ktir_cpu_b200 import check_status, kv_append, rotary_table
    gen = _gen(4)
    k, v = (_randn(gen, "f16", 3, 2, 64) for _ in range(2))
    kc, vc = (torch.zeros(2, 4, 2, 64, dtype=torch.float16, device="cuda") for _ in range(2))
    index = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    kv_append(k, v, kc, vc, index(0, 8, 1))
    with pytest.raises(IndexError):
        check_status()
    check_status()
    kv_append(k, v, kc, vc, index(4, 5, 6), positions=index(0, 10, -1), table=rotary_table(10, 64))
    with pytest.raises(IndexError):
        check_status()
    assert torch.equal(vc[1, 0], v[0]) and not vc[1, 1:].any()


# more tokens than blocks of one fit on the GPU at once, of few heads: several share a block
@pytest.mark.parametrize("typ,tokens,heads,kv_heads,dim,rot,page,interleaved,head_major", [
    ("bf16", 2003, 6, 1, 64, 64, 32, False, False),
    ("f16", 4001, 15, 3, 64, 32, 16, True, True),
    ("bf16", 2500, 1, 1, 16, 16, 1, False, False),
    ("f16", 1999, 2, 1, 256, 0, 8, False, False),
    ("bf16", 1801, 13, 5, 128, 128, 16, False, True),
])
def test_append_several_tokens_per_block(typ, tokens, heads, kv_heads, dim, rot, page, interleaved, head_major):
    test_append(typ, tokens, heads, kv_heads, dim, rot, page, interleaved, head_major)


def test_append_several_tokens_per_block_bad_indices():
    import torch
    from ktir_cpu_b200 import check_status, kv_append, rotary_table
    gen = _gen(5)
    k, v = (_randn(gen, "bf16", 2500, 1, 64) for _ in range(2))
    kc, vc = (torch.zeros(100, 25, 1, 64, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    slots = torch.arange(2500, dtype=torch.int32, device="cuda")
    positions = slots % 10
    bad = torch.tensor([0, 7, 1234, 2499], device="cuda")
    slots[bad[:2]] = 2500
    positions[bad[2]] = 10
    positions[bad[3]] = -1
    kv_append(k, v, kc, vc, slots, positions=positions, table=rotary_table(10, 64))
    with pytest.raises(IndexError):
        check_status()
    got = vc.reshape(2500, 1, 64)
    kept = torch.ones(2500, dtype=torch.bool, device="cuda")
    kept[bad] = False
    assert torch.equal(got[kept], v[kept]) and not got[bad].any() and not kc.reshape(2500, 64)[bad].any()


# -- decode -----------------------------------------------------------------------

def _decode_inputs(typ, lengths, heads, kv_heads, dim, page, head_major=False, seed=0, scale_q=1.0):
    import torch
    gen = _gen(seed)
    each = [-(-m // page) for m in lengths]
    total = sum(each) + 2
    kc, vc = (_cache(gen, typ, total, page, kv_heads, dim, head_major) for _ in range(2))
    order = torch.randperm(total, generator=gen, device="cuda").int().cpu()
    pages = torch.full((len(lengths), max(each + [1]) + 1), -7, dtype=torch.int32)
    at = 0
    for b, n in enumerate(each):
        pages[b, :n] = order[at:at + n]
        at += n
    q = (_randn(gen, typ, len(lengths), heads, dim).float() * scale_q).to(S.dtype_of(typ))
    return q, kc, vc, pages.cuda(), torch.tensor(lengths, dtype=torch.int32, device="cuda")


def _check_decode(typ, q, kc, vc, pages, lengths, scale, out, lse):
    S.decode(q, kc, vc, pages, lengths, scale,
             lambda b, hs, want: S.check_rows(f"seq {b} heads {hs}", out[b, hs], want, typ, q.shape[2], lse[b, hs]))


@pytest.mark.parametrize("typ,lengths,heads,kv_heads,dim,page,head_major", [
    ("bf16", [1], 4, 1, 128, 16, False),
    ("f16", [77], 32, 8, 128, 16, False),
    ("bf16", [0, 1, 15, 16, 17, 0, 63, 64, 65, 130], 8, 2, 64, 16, True),
    ("f16", [1000, 3, 257], 5, 5, 64, 24, False),
    ("bf16", [513, 40], 12, 4, 128, 1, True),
    ("f16", [70, 200], 48, 1, 128, 128, False),
    ("bf16", [300, 5], 34, 2, 64, 7, False),
    ("bf16", [9000], 8, 4, 128, 64, True),
    ("f16", [20000, 10, 0], 16, 2, 128, 32, False),
])
def test_decode(typ, lengths, heads, kv_heads, dim, page, head_major):
    from ktir_cpu_b200 import check_status, paged_decode
    x = _decode_inputs(typ, lengths, heads, kv_heads, dim, page, head_major, seed=sum(lengths))
    out, lse = paged_decode(*x, return_lse=True)
    check_status()
    _check_decode(typ, *x, dim ** -0.5, out, lse)


def test_decode_many_sequences():
    from ktir_cpu_b200 import check_status, paged_decode
    rng = random.Random(5)
    lengths = [rng.choice([0, 1, 2, 30, 64, 100, 300]) for _ in range(700)]
    x = _decode_inputs("bf16", lengths, 4, 2, 64, 16, seed=9)
    out, lse = paged_decode(*x, scale=0.3, return_lse=True)
    check_status()
    _check_decode("bf16", *x, 0.3, out, lse)


# how the keys are shared out: one sequence, whole or in parts; sequences with CTAs of their own, one or
# two to a lane that counts; too many tiles or too many sequences for that
@pytest.mark.parametrize("lengths", [
    [0], [1], [64], [256], [257], [384], [385], [1024], [1025], [30000],
    [640, 0, 65, 1000, 256, 257, 1, 3000],
    [130 + 37 * (b % 9) for b in range(32)],
    [(b * 61) % 300 for b in range(33)],
    [(b * 127) % 500 for b in range(64)],
    [1 + (b * 43) % 200 for b in range(65)],
    [3000 + 100 * b for b in range(20)],
    [0, 0] + [(b * 53) % 700 for b in range(90)] + [0] * 5,
    [769 * (b % 2) + b for b in range(150)],
    [768 - b for b in range(300)],
    [5000, 3, 0, 9],
])
@pytest.mark.parametrize("typ,heads,kv_heads,dim", [("bf16", 8, 2, 128), ("f16", 3, 1, 64), ("bf16", 32, 2, 64)])
def test_decode_shares_of_ctas(lengths, typ, heads, kv_heads, dim):
    from ktir_cpu_b200 import check_status, paged_decode
    x = _decode_inputs(typ, lengths, heads, kv_heads, dim, 16, seed=len(lengths))
    out, lse = paged_decode(*x, return_lse=True)
    again, lse2 = paged_decode(*x, return_lse=True)
    check_status()
    assert out.equal(again) and lse.equal(lse2)
    _check_decode(typ, *x, dim ** -0.5, out, lse)


@pytest.mark.parametrize("bad", [-3, 10 ** 6])
@pytest.mark.parametrize("batch", [1, 6, 40, 70])
def test_decode_bad_lengths(bad, batch):
    import torch
    from ktir_cpu_b200 import check_status, paged_decode
    x = _decode_inputs("bf16", [100 + 50 * b for b in range(batch)], 8, 2, 64, 16, seed=batch)
    lengths = x[-1].clone()
    lengths[batch // 2] = bad
    out, lse = paged_decode(*x[:-1], lengths, return_lse=True)
    with pytest.raises(IndexError):
        check_status()
    assert not out[batch // 2].any() and (lse[batch // 2] == -float("inf")).all()
    lengths[batch // 2] = 0
    _check_decode("bf16", *x[:-1], lengths, 64 ** -0.5, out, lse)
    check_status()


@pytest.mark.parametrize("typ", ["bf16", "f16"])
def test_decode_peaked_and_growing_scores(typ):
    """Scores in the hundreds, the largest at the end: the running maximum moves
    over and over, and most weights vanish."""
    import torch
    from ktir_cpu_b200 import check_status, paged_decode
    q, kc, vc, pages, lengths = _decode_inputs(typ, [700, 2000], 8, 2, 128, 16, seed=2, scale_q=4.0)
    ramp = torch.linspace(0.1, 3.0, 2000, device="cuda")
    for b, m in enumerate(lengths.tolist()):
        for i, p in enumerate(pages[b, :-(-m // 16)].tolist()):
            kc[p] = (kc[p].float() * ramp[16 * i:16 * i + 16, None, None]).to(kc.dtype)
    out, lse = paged_decode(q, kc, vc, pages, lengths, return_lse=True)
    check_status()
    _check_decode(typ, q, kc, vc, pages, lengths, 128 ** -0.5, out, lse)


def test_decode_ignores_what_lies_past_the_length():
    """Places past a sequence's length hold NaN and infinities."""
    import torch
    from ktir_cpu_b200 import check_status, paged_decode
    q, kc, vc, pages, lengths = _decode_inputs("f16", [5, 33, 100, 0], 8, 2, 128, 32, seed=6)
    clean = paged_decode(q, kc, vc, pages, lengths)
    used = torch.zeros(kc.shape[:2], dtype=torch.bool, device="cuda")
    for b, m in enumerate(lengths.tolist()):
        for j in range(m):
            used[int(pages[b, j // 32]), j % 32] = True
    for i, bad in enumerate([math.nan, math.inf, -math.inf]):
        kc[~used], vc[~used] = bad, bad
        assert torch.equal(paged_decode(q, kc, vc, pages, lengths), clean), bad
    check_status()


def test_decode_strides_streams_and_repeats():
    """Strided queries and outputs, another stream, calls of different sizes in turn,
    and the same result every time."""
    import torch
    from ktir_cpu_b200 import check_status, paged_decode
    small = _decode_inputs("bf16", [40, 900], 8, 2, 128, 16, seed=11)
    large = _decode_inputs("bf16", [5000, 100, 7, 3000], 16, 4, 128, 16, seed=12)
    a, b = paged_decode(*small), paged_decode(*large)
    wide = torch.zeros(2, 8, 3, 128, dtype=torch.bfloat16, device="cuda")
    wide[:, :, 1] = small[0]
    into = torch.zeros_like(wide)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    for _ in range(20):
        got = paged_decode(wide[:, :, 1], *small[1:], out=into[:, :, 2])
        assert torch.equal(got, a) and not into[:, :, :2].any()
        with torch.cuda.stream(stream):
            other = paged_decode(*large)
        stream.synchronize()
        assert torch.equal(other, b) and torch.equal(paged_decode(*large), b)
    check_status()


def test_decode_in_a_graph():
    import torch
    from ktir_cpu_b200 import check_status, paged_decode
    x = _decode_inputs("bf16", [3000, 17, 400], 16, 4, 128, 16, seed=13)
    want = paged_decode(*x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = paged_decode(*x)
    for _ in range(3):
        got.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)
    x[4][1] = 5
    graph.replay()
    assert torch.equal(got, paged_decode(*x))
    check_status()


def test_decode_reports_bad_indices():
    from ktir_cpu_b200 import check_status, paged_decode
    for at, bad in [((3, (0, 1)), -1), ((3, (0, 1)), 1 << 20), ((4, (0,)), 500), ((4, (0,)), -3)]:
        x = _decode_inputs("bf16", [40, 20], 4, 2, 64, 16, seed=14)
        x[at[0]][at[1]] = bad
        out, lse = paged_decode(*x, return_lse=True)
        with pytest.raises(IndexError):
            check_status()
        # the other sequence is not touched by it (how it is split may be)
        _check_decode("bf16", x[0][1:], x[1], x[2], x[3][1:], x[4][1:], 64 ** -0.5, out[1:], lse[1:])


def test_decode_past_32_bits():
    """Element offsets above 2^31 in the cache."""
    import torch
    from ktir_cpu_b200 import check_status, paged_decode
    pages, page, hk, d = 66000, 16, 16, 128            # 2.16e9 elements, 4.3 GB each
    kc, vc = (torch.zeros(pages, page, hk, d, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    gen = _gen(15)
    last = [65999, 65990, 3]
    for p in last:
        kc[p], vc[p] = _randn(gen, "bf16", page, hk, d), _randn(gen, "bf16", page, hk, d)
    q = _randn(gen, "bf16", 1, 16, d)
    table = torch.tensor([last], dtype=torch.int32, device="cuda")
    lengths = torch.tensor([41], dtype=torch.int32, device="cuda")
    out, lse = paged_decode(q, kc, vc, table, lengths, return_lse=True)
    check_status()
    _check_decode("bf16", q, kc, vc, table, lengths, d ** -0.5, out, lse)


# -- prompt -----------------------------------------------------------------------

def _prompt_inputs(typ, new, keys, heads, kv_heads, dim, seed=0):
    import torch
    gen = _gen(seed)
    q = _randn(gen, typ, sum(new), heads, dim)
    kv = _randn(gen, typ, sum(keys), 2 * kv_heads, dim)
    ends = lambda each: torch.tensor([0] + each, device="cuda").cumsum(0).int()  # noqa: E731
    return q, kv[:, :kv_heads], kv[:, kv_heads:], ends(new), ends(keys)


def _check_prompt(typ, q, k, v, offsets, kv_offsets, causal, scale, out, lse):
    S.prompt(q, k, v, offsets, kv_offsets, causal, scale,
             lambda ts, h, want: S.check_rows(f"tokens {ts} head {h}", out[ts, h], want, typ, q.shape[2], lse[ts, h]))


@pytest.mark.parametrize("typ,new,keys,heads,kv_heads,dim,causal", [
    ("bf16", [1], [1], 4, 1, 128, True),
    ("f16", [19], [19], 32, 8, 128, True),
    ("bf16", [0, 1, 127, 128, 129, 0, 255, 257, 0], None, 4, 2, 128, True),
    ("f16", [300, 31, 64, 2], None, 5, 5, 64, True),
    ("bf16", [200, 40], None, 12, 2, 64, False),
    ("f16", [130, 77], None, 7, 1, 128, False),
    ("bf16", [33, 5, 0, 100], [500, 5, 64, 101], 6, 2, 128, True),
    ("f16", [17, 1, 20], [300, 129, 900], 3, 1, 64, True),
    ("bf16", [50, 200, 9], [20, 60, 0], 4, 2, 64, True),      # rows that see no key
    ("f16", [50, 9], [20, 0], 4, 2, 128, False),
    ("bf16", [1030], None, 2, 1, 128, True),
    ("bf16", [70, 3], None, 80, 1, 128, True),
    ("f16", [5, 260], None, 128, 1, 64, True),
    ("bf16", [2100, 600], None, 3, 3, 64, True),
])
def test_prompt(typ, new, keys, heads, kv_heads, dim, causal):
    from ktir_cpu_b200 import check_status, prompt_attention
    q, k, v, offsets, kv_offsets = _prompt_inputs(typ, new, keys or new, heads, kv_heads, dim, seed=sum(new))
    out, lse = prompt_attention(q, k, v, offsets, kv_offsets=kv_offsets if keys else None, causal=causal,
                                return_lse=True)
    check_status()
    _check_prompt(typ, q, k, v, offsets, kv_offsets, causal, dim ** -0.5, out, lse)


@pytest.mark.parametrize("typ,new,keys,heads,kv_heads,dim,causal", [
    ("bf16", [64], [8192], 32, 8, 128, True),
    ("f16", [16] * 4, [5000] * 4, 8, 2, 64, True),
    ("bf16", [3, 70, 0, 1], [3000, 2001, 50, 4096], 6, 2, 128, True),
    ("f16", [40, 100], [6000, 30], 4, 4, 128, False),
    ("bf16", [200], [40], 2, 1, 64, True),
    ("bf16", [1, 1], [20000, 7], 16, 1, 128, True),
])
def test_prompt_few_queries_over_many_keys(typ, new, keys, heads, kv_heads, dim, causal):
    """The keys of a few queries are shared among the SMs; the same result every time."""
    import torch
    from ktir_cpu_b200 import check_status, prompt_attention
    q, k, v, offsets, kv_offsets = _prompt_inputs(typ, new, keys, heads, kv_heads, dim, seed=sum(keys))
    out, lse = prompt_attention(q, k, v, offsets, kv_offsets=kv_offsets, causal=causal, return_lse=True)
    _check_prompt(typ, q, k, v, offsets, kv_offsets, causal, dim ** -0.5, out, lse)
    for _ in range(50):
        again, lse2 = prompt_attention(q, k, v, offsets, kv_offsets=kv_offsets, causal=causal, return_lse=True)
        assert torch.equal(again, out) and torch.equal(lse2, lse)
    check_status()


def test_prompt_many_tiles_of_many_keys():
    """More weights of tiles than a table of them holds: some of the heads, all tokens."""
    import torch
    from ktir_cpu_b200 import check_status, prompt_attention
    q, k, v, offsets, kv_offsets = _prompt_inputs("f16", [700, 9], [45000, 9], 128, 1, 64, seed=41)
    out, lse = prompt_attention(q, k, v, offsets, kv_offsets=kv_offsets, return_lse=True)
    check_status()
    for h in (0, 77):
        _check_prompt("f16", q[:, h:h + 1], k, v, offsets, kv_offsets, True, 0.125, out[:, h:h + 1], lse[:, h:h + 1])


def test_prompt_mixed_calls_in_turn():
    """Calls that split keys, take row tiles singly and in pairs, one after the other."""
    import torch
    from ktir_cpu_b200 import check_status, prompt_attention
    calls = []
    for i, (new, keys) in enumerate([([64], [4000]), ([30] * 100, [30] * 100), ([700] * 9, [700] * 9), ([5], [900]),
                                     ([81, 33, 300] * 5, [400] * 15)]):
        q, k, v, offsets, kv_offsets = _prompt_inputs("bf16", new, keys, 8, 2, 128, seed=30 + i)
        first, lse = prompt_attention(q, k, v, offsets, kv_offsets=kv_offsets, return_lse=True)
        _check_prompt("bf16", q, k, v, offsets, kv_offsets, True, 128 ** -0.5, first, lse)
        calls.append((q, k, v, offsets, kv_offsets, first))
    for _ in range(20):
        outs = [prompt_attention(*c[:4], kv_offsets=c[4]) for c in calls]
        assert all(torch.equal(o, c[5]) for o, c in zip(outs, calls))
    check_status()


def test_prompt_many_short():
    from ktir_cpu_b200 import check_status, prompt_attention
    rng = random.Random(8)
    new = [rng.choice([0, 1, 2, 5, 17, 40]) for _ in range(500)]
    x = _prompt_inputs("bf16", new, new, 2, 1, 64, seed=16)
    out, lse = prompt_attention(*x[:4], scale=0.2, return_lse=True)
    check_status()
    _check_prompt("bf16", *x, True, 0.2, out, lse)


# few row tiles: a CTA's halves of the keys, around the blocks (80 keys at dim 128, 128 at dim 64) where that begins
@pytest.mark.parametrize("keys", [160, 161, 240, 241, 256, 257, 320, 385, 1280, 1281])
@pytest.mark.parametrize("typ,new,heads,kv_heads,dim,causal", [
    ("bf16", 5, 4, 2, 128, True),
    ("f16", 130, 3, 1, 64, True),
    ("f16", 40, 6, 6, 128, False),
    ("bf16", 300, 2, 2, 64, True),        # more queries than some have keys: rows that see none
])
def test_prompt_halves_of_keys(keys, typ, new, heads, kv_heads, dim, causal):
    from ktir_cpu_b200 import check_status, prompt_attention
    q, k, v, offsets, kv_offsets = _prompt_inputs(typ, [new], [keys], heads, kv_heads, dim, seed=keys)
    out, lse = prompt_attention(q, k, v, offsets, kv_offsets=kv_offsets, causal=causal, return_lse=True)
    check_status()
    _check_prompt(typ, q, k, v, offsets, kv_offsets, causal, dim ** -0.5, out, lse)


@pytest.mark.parametrize("typ,dim", [("bf16", 128), ("f16", 64), ("f16", 128)])
@pytest.mark.parametrize("rising", [True, False])
def test_prompt_peaked_scores(typ, dim, rising):
    """Large scores, rising or falling along the keys: the running maximum moves
    over and over, or most later weights vanish."""
    import torch
    from ktir_cpu_b200 import check_status, prompt_attention
    q, k, v, offsets, kv_offsets = _prompt_inputs(typ, [900, 300], [900, 300], 4, 2, dim, seed=17)
    ramp = torch.linspace(0.1, 6.0, 1200, device="cuda")
    k = (k.float() * (ramp if rising else ramp.flip(0))[:, None, None]).to(k.dtype)
    out, lse = prompt_attention(q, k, v, offsets, return_lse=True)
    check_status()
    _check_prompt(typ, q, k, v, offsets, kv_offsets, True, dim ** -0.5, out, lse)


def test_prompt_sequences_do_not_mix():
    """NaN and infinities in one sequence reach no other."""
    import torch
    from ktir_cpu_b200 import check_status, prompt_attention
    new = [70, 33, 150, 20]
    q, k, v, offsets, _ = _prompt_inputs("bf16", new, new, 4, 2, 128, seed=18)
    clean = prompt_attention(q, k, v, offsets)
    for bad in [math.nan, math.inf, -math.inf]:
        for lo, hi in [(0, 70), (103, 253)]:
            q2, k2, v2 = q.clone(), k.clone(), v.clone()
            q2[lo:hi], k2[lo:hi], v2[lo:hi] = bad, bad, bad
            got = prompt_attention(q2, k2, v2, offsets)
            assert torch.equal(got[:lo], clean[:lo]) and torch.equal(got[hi:], clean[hi:]), (bad, lo)
    check_status()


def test_prompt_infinite_keys_in_masked_places():
    """A later key that is infinite or NaN moves no earlier row."""
    import torch
    from ktir_cpu_b200 import check_status, prompt_attention
    q, k, v, offsets, _ = _prompt_inputs("bf16", [200], [200], 4, 2, 128, seed=19)
    clean = prompt_attention(q, k, v, offsets)
    for bad in [math.nan, math.inf]:
        k2 = k.clone()
        k2[150:] = bad
        got = prompt_attention(q, k2, v, offsets)
        assert torch.equal(got[:150], clean[:150])
    check_status()


def test_prompt_strides_out_and_graph():
    import torch
    from ktir_cpu_b200 import check_status, prompt_attention
    q, k, v, offsets, kv_offsets = _prompt_inputs("f16", [140, 61], [140, 61], 6, 2, 64, seed=20)
    want = prompt_attention(q, k, v, offsets)
    # head-major memory, and outputs inside a larger buffer
    q2, k2, v2 = (x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v))
    into = torch.zeros(201, 8, 128, dtype=torch.float16, device="cuda")
    got = prompt_attention(q2, k2, v2, offsets, out=into[:, 1:7, 64:])
    assert torch.equal(got, want)
    assert not into[:, 0].any() and not into[:, 7].any() and not into[:, :, :64].any()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        again = prompt_attention(q, k, v, offsets)
    for _ in range(3):
        again.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(again, want)
    # keys and values that all heads of a broadcast input share
    one = k[:, :1].expand(-1, 2, -1)
    assert torch.equal(prompt_attention(q, one, one, offsets),
                       prompt_attention(q, one.contiguous(), one.contiguous(), offsets))
    check_status()


def test_prompt_reports_bad_offsets():
    import torch
    from ktir_cpu_b200 import check_status, prompt_attention
    q, k, v, offsets, kv_offsets = _prompt_inputs("bf16", [40, 30], [50, 60], 2, 1, 64, seed=21)
    for bad in ([0, 50, 111], [0, 50, 40], [-1, 50, 110]):
        prompt_attention(q, k, v, offsets, kv_offsets=torch.tensor(bad, dtype=torch.int32, device="cuda"))
        with pytest.raises(IndexError):
            check_status()
    prompt_attention(q, k, v, offsets, kv_offsets=kv_offsets)
    check_status()


# -- refusals with tensors on the GPU, and the pieces together ------------------------

def test_refusals():
    import torch
    from ktir_cpu_b200 import kv_append, paged_decode, prompt_attention
    q, kc, vc, pages, lengths = _decode_inputs("bf16", [40, 20], 4, 2, 64, 16, seed=22)
    off = torch.tensor([0, 2], dtype=torch.int32, device="cuda")
    k = kc[0, :2]
    slots = off
    for call, kind in [
        (lambda: paged_decode(q.float(), kc, vc, pages, lengths), NotImplementedError),
        (lambda: paged_decode(q, kc.half(), vc, pages, lengths), ValueError),
        (lambda: paged_decode(q[:, :3], kc, vc, pages, lengths), ValueError),
        (lambda: paged_decode(q, kc, vc, pages.long(), lengths), ValueError),
        (lambda: paged_decode(q, kc, vc, pages, lengths[:1]), ValueError),
        (lambda: paged_decode(q, kc, vc, pages, lengths.cpu()), ValueError),
        (lambda: paged_decode(q, kc, vc, pages, lengths, scale=-1.0), NotImplementedError),
        (lambda: paged_decode(q, kc, vc, pages, lengths, scale=math.nan), NotImplementedError),
        (lambda: paged_decode(q[..., :32], kc[..., :32], vc[..., :32], pages, lengths), NotImplementedError),
        (lambda: paged_decode(q.requires_grad_(), kc, vc, pages, lengths), RuntimeError),
        (lambda: paged_decode(torch.zeros(2, 4, 65, dtype=q.dtype, device="cuda")[..., 1:], kc, vc, pages, lengths),
         NotImplementedError),
        (lambda: prompt_attention(k, k, k[:1], off), ValueError),
        (lambda: prompt_attention(k, k[:1], k[:1], off), ValueError),
        (lambda: prompt_attention(k, k, k, off[:1]), ValueError),
        (lambda: prompt_attention(k, k, k, off, kv_offsets=off[:1]), ValueError),
        (lambda: prompt_attention(k, k, k, off, out=k[:1]), ValueError),
        (lambda: prompt_attention(k.transpose(1, 2), k, k, off), NotImplementedError),
        (lambda: kv_append(k, k[:1], kc, vc, slots), ValueError),
        (lambda: kv_append(k, k, kc, vc[:1], slots), ValueError),
        (lambda: kv_append(k, k, kc, vc, slots.long()), ValueError),
        (lambda: kv_append(k, k, kc, vc, slots, positions=slots), ValueError),
        (lambda: kv_append(k, k, kc, vc, slots, positions=slots, table=torch.zeros(8, 24, device="cuda")),
         NotImplementedError),
        (lambda: kv_append(k, k, kc, vc, slots, q_out=k), ValueError),
    ]:
        with pytest.raises(kind):
            call()
        q.requires_grad_(False)


def test_empty_calls():
    import torch
    from ktir_cpu_b200 import check_status, kv_append, paged_decode, prompt_attention
    e = torch.zeros(0, 4, 64, dtype=torch.bfloat16, device="cuda")
    c = torch.zeros(3, 8, 2, 64, dtype=torch.bfloat16, device="cuda")
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    assert paged_decode(e, c, c, none.view(0, 0), none).shape == (0, 4, 64)
    off = torch.zeros(3, dtype=torch.int32, device="cuda")
    assert prompt_attention(e, e[:, :2], e[:, :2], off).shape == (0, 4, 64)
    kv_append(e[:, :2], e[:, :2], c, c.clone(), none)
    check_status()


def test_prompt_then_decode_agree():
    """A prompt read in one pass, and the same tokens one at a time over the cache."""
    import torch
    from ktir_cpu_b200 import check_status, kv_append, paged_decode, prompt_attention, rotary_table
    gen = _gen(23)
    n, heads, kv_heads, dim, page = 70, 8, 2, 128, 16
    q, k, v = _randn(gen, "bf16", n, heads, dim), _randn(gen, "bf16", n, kv_heads, dim), _randn(gen, "bf16", n, kv_heads, dim)
    kc, vc = (torch.zeros(6, page, kv_heads, dim, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    pages = torch.tensor([[4, 0, 5, 2, 1]], dtype=torch.int32, device="cuda")
    at = torch.arange(n, device="cuda")
    slots = (pages[0].long()[at // page] * page + at % page).int()
    args = dict(table=rotary_table(128, dim))
    turned = kv_append(k, v, kc, vc, slots, q=q, positions=at.int(), **args)
    keys = kc[slots.long() // page, slots.long() % page]
    whole = prompt_attention(turned, keys, v, torch.tensor([0, n], dtype=torch.int32, device="cuda"))
    # each side: one rounding of the output and one of the weights, both relative to at most max |v|
    bound = 2 * 2 * S.U["bf16"] * float(v.abs().max()) * 1.01
    for i in range(n):
        one = paged_decode(turned[i:i + 1], kc, vc, pages, torch.tensor([i + 1], dtype=torch.int32, device="cuda"))
        assert (one[0].double() - whole[i].double()).abs().max() <= bound
    check_status()


# -- scores far from 0 ---------------------------------------------------------------

def _far(typ, keys, dim, best):
    """Integer vectors: every score is exact in 32 bits, key `best`'s the largest by
    more than 2^20, and its product with scale log2(e) is not."""
    import torch
    q = torch.full((1, 1, dim), 3 * 4096., device="cuda").to(S.dtype_of(typ))
    k = torch.full((keys, 1, dim), 1024., device="cuda").to(S.dtype_of(typ))
    k[best] = 5 * 4096.
    return q, k, _randn(_gen(keys), typ, keys, 1, dim)


@pytest.mark.parametrize("typ", ["bf16", "f16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("keys,best", [(1, 0), (90, 3), (300, 0), (300, 150), (3000, 2999)])
@pytest.mark.parametrize("scale", [None, 0.1, 0.3])
def test_far_scores(typ, dim, keys, best, scale):
    """One score stands out by so much that every other weight is below 2^-1000: the
    output is that key's value, to the bit."""
    import torch
    from ktir_cpu_b200 import check_status, paged_decode, prompt_attention
    q, k, v = _far(typ, keys, dim, best)
    for sign in (1, -1):           # the largest score of all, or the others far below 0
        qs, ks = (q, k) if sign > 0 else (-q, torch.where(k == k[best], 1.0, 5 * 4096.).to(k.dtype))
        if keys == 1:
            ks = k
        ends = torch.tensor([0, 1, keys], dtype=torch.int32, device="cuda")
        out = prompt_attention(qs, ks, v, ends[:2], kv_offsets=ends[::2].contiguous(), scale=scale)
        assert torch.equal(out[0, 0], v[best, 0])
        pages = torch.arange(keys, dtype=torch.int32, device="cuda")[None]
        out = paged_decode(qs, ks[:, None], v[:, None], pages, ends[2:], scale=scale)
        assert torch.equal(out[0, 0], v[best, 0])
    check_status()


@pytest.mark.parametrize("typ", ["bf16", "f16"])
@pytest.mark.parametrize("size", [3000.0, 9000.0])
def test_far_scores_close_together(typ, size):
    """Scores of 2^27 and more, a few units apart: how the weights fall is open within
    the scores' own rounding, but they sum to 1.  With values of 1, each output is a sum
    of weights rounded to the element type over the sum of the unrounded ones, then
    rounded: 1 within two unit roundoffs, the sums' 2 n 2^-24 and, in f16, 2^-25 for each
    weight below the normal range."""
    import torch
    from ktir_cpu_b200 import check_status, paged_decode, prompt_attention
    n, dim = 500, 64
    gen = _gen(int(size))
    base = torch.randn(1, 1, dim, generator=gen, device="cuda").sign() * size
    q = base.expand(n, 4, dim).to(S.dtype_of(typ))
    k = base.expand(n, 1, dim).to(S.dtype_of(typ)).clone()
    k[torch.arange(n, device="cuda"), 0, torch.arange(n, device="cuda") % dim] = 0
    v = torch.ones(n, 1, dim, dtype=k.dtype, device="cuda")
    bound = 2 * S.U[typ] + 2 * n * S.E + (n * 2.0 ** -25 if typ == "f16" else 0.0)
    ends = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    for scale in (0.3, 0.1, 1.0):
        for keys in (k, k * torch.linspace(0.99, 1.01, n, device="cuda")[:, None, None].to(k.dtype)):
            out = prompt_attention(q, keys, v, ends, scale=scale).double()
            assert ((out - 1).abs() <= bound).all()
            pages = torch.arange(n, dtype=torch.int32, device="cuda")[None]
            out = paged_decode(q[:1], keys[:, None], v[:, None], pages, ends[1:], scale=scale).double()
            assert ((out - 1).abs() <= bound).all()
    check_status()


# -- sizes of zero ---------------------------------------------------------------------

def test_append_without_heads():
    """Queries without heads: keys and values are written all the same.  Keys without
    heads are refused: no output is returned that nothing wrote."""
    import torch
    from ktir_cpu_b200 import check_status, kv_append
    gen = _gen(50)
    k, v = _randn(gen, "bf16", 3, 2, 64), _randn(gen, "bf16", 3, 2, 64)
    kc, vc = (torch.zeros(2, 4, 2, 64, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    slots = torch.tensor([5, 0, 2], dtype=torch.int32, device="cuda")
    out = kv_append(k, v, kc, vc, slots, q=k[:, :0])
    assert out.shape == (3, 0, 64)
    assert torch.equal(kc.flatten(0, 1)[slots.long()], k) and torch.equal(vc.flatten(0, 1)[slots.long()], v)
    with pytest.raises(ValueError, match="no heads"):
        kv_append(k[:, :0], v[:, :0], kc[:, :, :0], vc[:, :, :0], slots, q=k)
    check_status()


def _fill_free_memory(value=7.0):
    """Whatever is allocated next holds `value` until something is written."""
    import torch
    for n in (10, 14, 18, 22):
        blocks = [torch.full((1 << n,), value, dtype=torch.bfloat16, device="cuda") for _ in range(8)]
        del blocks


@pytest.mark.parametrize("tokens,kv_heads", [(6, 2), (2500, 1)])       # one token per block, and several
@pytest.mark.parametrize("rot", [0, 32, 64])
def test_append_bad_indices_leave_no_row_unwritten(tokens, kv_heads, rot):
    """A query does not depend on its token's slot; one without a position is zero."""
    import torch
    from ktir_cpu_b200 import check_status, kv_append, rotary_table
    gen = _gen(51)
    q, k, v = (_randn(gen, "bf16", tokens, kv_heads, 64) for _ in range(3))
    page = 25
    kc, vc = (torch.zeros(tokens // page + 1, page, kv_heads, 64, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    slots = torch.arange(tokens, dtype=torch.int32, device="cuda")
    positions = slots % 10
    args = dict(positions=positions, table=rotary_table(10, rot)) if rot else {}
    want = kv_append(k, v, kc.clone(), vc.clone(), slots, q=q, **args)
    check_status()

    # padding without a position: nothing to report
    slots[1], slots[2], positions[2] = -1, -1, -1
    _fill_free_memory()
    got = kv_append(k, v, kc, vc, slots, q=q, **args)
    check_status()
    if rot:
        assert not got[2].any()
    same = torch.ones(tokens, dtype=torch.bool, device="cuda")
    same[2] = not rot
    assert torch.equal(got[same], want[same])

    slots[0] = kc.shape[0] * page                   # past the cache
    positions[3], positions[4] = 10, -1             # not in the table
    kc.zero_(), vc.zero_()
    _fill_free_memory()
    got = kv_append(k, v, kc, vc, slots, q=q, **args)
    with pytest.raises(IndexError):
        check_status()
    if rot:
        assert not got[2:5].any()
        same[3:5] = False
    assert torch.equal(got[same], want[same])
    written = same & (slots >= 0)
    written[0] = False
    assert torch.equal(vc.flatten(0, 1)[:tokens][written], v[written])
    assert not vc.flatten(0, 1)[:tokens][~written].any() and not kc.flatten(0, 1)[:tokens][~written].any()


@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 2, 128), (3, 1, 64), (64, 2, 64)])
@pytest.mark.parametrize("offsets,kv_offsets,valid", [
    ([0, 50, 111], [0, 60, 110], [0]),               # past the tokens
    ([0, 50, 20, 100], [0, 60, 80, 110], []),        # falling: rows 20 to 49 are two sequences', either may stay
    ([-1, 50, 100], [0, 60, 110], [1]),
    ([0, 50, 100], [0, 60, 300], [0]),               # keys past their tokens
    ([0, 50, 100], [0, 120, 110], []),
    ([7, 50, 90], [0, 60, 110], [0, 1]),             # tokens before the first sequence and after the last
    ([0, 0, 0], [0, 60, 110], []),
])
def test_prompt_bad_offsets_leave_no_row_unwritten(heads, kv_heads, dim, offsets, kv_offsets, valid):
    import torch
    from ktir_cpu_b200 import check_status, prompt_attention
    q, k, v, _, _ = _prompt_inputs("bf16", [100], [110], heads, kv_heads, dim, seed=52)
    index = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    _fill_free_memory()
    out, lse = prompt_attention(q, k, v, index(offsets), kv_offsets=index(kv_offsets), return_lse=True)
    with pytest.raises(IndexError):
        check_status()
    free = torch.ones(100, dtype=torch.bool, device="cuda")
    for b, (lo, hi, k0, k1) in enumerate(zip(offsets, offsets[1:], kv_offsets, kv_offsets[1:])):
        if 0 <= lo <= hi <= 100 and 0 <= k0 <= k1 <= 110:
            free[lo:hi] = False
        if b in valid:
            _check_prompt("bf16", q[lo:hi], k[k0:k1], v[k0:k1], index([0, hi - lo]), index([0, k1 - k0]), True,
                          dim ** -0.5, out[lo:hi], lse[lo:hi])
    assert not out[free].any() and (lse[free] == -math.inf).all()
    check_status()


@pytest.mark.parametrize("first", [True, False])      # the largest weight's key
@pytest.mark.parametrize("heads", [1, 160, 600])      # shared out over the keys, and not
@pytest.mark.parametrize("dim", [64, 128])
def test_f16_many_small_weights(dim, heads, first):
    """131,071 keys of weight 2^-25.5 beside one of weight 1: 0.0028 of the sum, each
    weight below what f16 holds next to 1.  A weight is good to 2^-32 of the largest."""
    import torch
    from ktir_cpu_b200 import check_status, paged_decode, prompt_attention
    n, page = 131072, 64
    at = 0 if first else n - 1
    q = torch.zeros(1, heads, dim, dtype=torch.float16, device="cuda")
    q[..., 0] = 1
    k = torch.zeros(n, 1, dim, dtype=torch.float16, device="cuda")
    k[..., 0] = -25.5
    k[at] = 0
    v = torch.ones_like(k)
    v[at] = 0
    scale = math.log(2.0)
    small = (n - 1) * 2.0 ** -25.5
    want = small / (1 + small)
    score = (dim + 4) * S.E * 25.5 * scale + 2.0 ** -21
    bound = S.U["f16"] * want + (S.U["f16"] + 2 * score + 2 * S.E * n) * want + 2.0 ** -32 * n + 2.0 ** -25
    lim = score + S.E * n + 2 * S.E
    ends = torch.tensor([0, 1, n], dtype=torch.int32, device="cuda")
    shared = lambda x: x.expand(-1, heads, -1)  # noqa: E731
    out, lse = prompt_attention(q, shared(k), shared(v), ends[:2], kv_offsets=ends[::2].contiguous(), scale=scale,
                                return_lse=True)
    assert ((out.double() - want).abs() <= bound).all(), float((out.double() - want).abs().max() / bound)
    assert ((lse.double() - math.log1p(small)).abs() <= lim).all()
    paged = lambda x: x.view(n // page, page, 1, dim).expand(-1, -1, heads, -1)  # noqa: E731
    out, lse = paged_decode(q, paged(k), paged(v), torch.arange(n // page, dtype=torch.int32, device="cuda")[None],
                            ends[2:], scale=scale, return_lse=True)
    assert ((out.double() - want).abs() <= bound).all(), float((out.double() - want).abs().max() / bound)
    assert ((lse.double() - math.log1p(small)).abs() <= lim).all()
    check_status()


def test_workspaces_after_a_reported_timeout():
    """The status word as a wait that ran out leaves it: the kept workspaces go, and the
    next calls, split and not, are right."""
    import torch
    from ktir_cpu_b200 import check_status, paged_decode, prompt_attention, runtime, serving
    q, k, v, offsets, kv_offsets = _prompt_inputs("bf16", [64], [8192], 8, 2, 128, seed=53)
    x = _decode_inputs("bf16", [3000, 40], 8, 2, 128, 16, seed=53)
    want, want2 = prompt_attention(q, k, v, offsets, kv_offsets=kv_offsets), paged_decode(*x)
    check_status()
    device = torch.cuda.current_device()
    before = torch.cuda.memory_allocated()
    serving._ext().status(device).fill_(runtime.STATUS_TIMEOUT)
    with pytest.raises(RuntimeError, match="timed out"):
        check_status()
    # parts of both operators: 16 rows of 130 floats twice for 512 CTAs, 128 rows of 130 for 160
    assert before - torch.cuda.memory_allocated() >= 4 * 130 * (512 * 2 * 16 + 160 * 128)
    for _ in range(3):
        assert torch.equal(prompt_attention(q, k, v, offsets, kv_offsets=kv_offsets), want)
        assert torch.equal(paged_decode(*x), want2)
    check_status()


def test_gradients_and_tangents_are_refused():
    """Neither a gradient nor a forward-mode tangent is lost without a word."""
    import torch
    import torch.autograd.forward_ad as fw
    from ktir_cpu_b200 import check_status, kv_append, paged_decode, prompt_attention, rotary_table
    q, kc, vc, pages, lengths = _decode_inputs("bf16", [40, 20], 4, 2, 64, 16, seed=54)
    k, v = kc[0, :2].clone(), vc[0, :2].clone()
    off = torch.tensor([0, 2], dtype=torch.int32, device="cuda")
    table = rotary_table(8, 64)
    calls = {
        "append": lambda q, k, v, kc, vc, t: kv_append(k, v, kc, vc, off, q=q, positions=off, table=t),
        "decode": lambda q, k, v, kc, vc, t: paged_decode(q, kc, vc, pages, lengths),
        "prompt": lambda q, k, v, kc, vc, t: prompt_attention(q, k, v, off),
    }
    takes = {"append": (0, 1, 2, 3, 4, 5), "decode": (0, 3, 4), "prompt": (0, 1, 2)}
    for name, call in calls.items():
        for at in takes[name]:
            args = [q, k, v, kc, vc, table]
            with fw.dual_level():
                args[at] = fw.make_dual(args[at], torch.ones_like(args[at]))
                with pytest.raises(RuntimeError, match="tangent"):
                    call(*args)
                with fw._set_fwd_grad_enabled(False):
                    call(*args)
            args[at] = [q, k, v, kc, vc, table][at].clone().requires_grad_()
            with pytest.raises(RuntimeError, match="gradient"):
                call(*args)
            with torch.no_grad():
                call(*args)
    check_status()


def test_written_tensors_are_seen_as_changed():
    """Caches and given outputs count as written in place, inputs do not; a tensor saved
    for a gradient and written since is found out."""
    import torch
    from ktir_cpu_b200 import check_status, kv_append, paged_decode, prompt_attention
    q, kc, vc, pages, lengths = _decode_inputs("bf16", [40, 20], 4, 2, 64, 16, seed=55)
    k, v = kc[0, :2].clone(), vc[0, :2].clone()
    off = torch.tensor([0, 2], dtype=torch.int32, device="cuda")
    out, q_out = torch.empty_like(q), torch.empty_like(q)
    read, write = (q, k, v, pages, lengths, off), (kc, vc, q_out, out)
    for call, moves in [(lambda: kv_append(k, v, kc, vc, off, q=q, q_out=q_out), (1, 1, 1, 0)),
                        (lambda: kv_append(k, v, kc, vc, off), (1, 1, 0, 0)),
                        (lambda: paged_decode(q, kc, vc, pages, lengths, out=out), (0, 0, 0, 1)),
                        (lambda: prompt_attention(q, k, v, off, out=out), (0, 0, 0, 1))]:
        was_read, was = [t._version for t in read], [t._version for t in write]
        call()
        assert [t._version for t in read] == was_read
        assert [t._version - w for t, w in zip(write, was)] == list(moves)
    weight = torch.ones(64, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    loss = (kc * weight).sum()
    kv_append(k, v, kc, vc, off)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    with torch.inference_mode():
        c = torch.zeros_like(kc)
        kv_append(k, v, c, c.clone(), off)
    kv_append(k, v, c, c.clone(), off)              # inference tensors keep no count
    check_status()


def test_outputs_that_share_memory_are_refused():
    import torch
    from ktir_cpu_b200 import check_status, kv_append, paged_decode, prompt_attention
    q, kc, vc, pages, lengths = _decode_inputs("bf16", [40, 20], 4, 2, 64, 16, seed=56)
    k, v = kc[0, :2].clone(), vc[0, :2].clone()
    off = torch.tensor([0, 2], dtype=torch.int32, device="cuda")
    for call in [lambda: paged_decode(q, kc, vc, pages, lengths, out=q[:1].clone().expand(2, -1, -1)),
                 lambda: prompt_attention(q, k, v, off, out=q[:, :1].clone().expand(-1, 4, -1)),
                 lambda: kv_append(k, v, kc, vc, off, q=q, q_out=q[:1].clone().expand(2, -1, -1)),
                 lambda: kv_append(k, v, kc[:1].expand(9, -1, -1, -1), vc[:1].expand(9, -1, -1, -1), off)]:
        with pytest.raises(ValueError, match="share memory"):
            call()
    one = q[:1].clone()
    assert torch.equal(paged_decode(q[:1], kc, vc, pages[:1], lengths[:1], out=one.as_strided((1, 4, 64), (0, 64, 1))),
                       paged_decode(q[:1], kc, vc, pages[:1], lengths[:1]))
    check_status()


# -- captured calls ------------------------------------------------------------------

def _nodes(graph):
    """(kernels, bytes cleared, other nodes) of a captured graph."""
    import ctypes as C
    rt = C.CDLL("libcudart.so.12")

    class Memset(C.Structure):
        _fields_ = [("dst", C.c_void_p), ("pitch", C.c_size_t), ("value", C.c_uint), ("element", C.c_uint),
                    ("width", C.c_size_t), ("height", C.c_size_t)]

    raw, n = C.c_void_p(graph.raw_cuda_graph()), C.c_size_t(0)
    assert rt.cudaGraphGetNodes(raw, None, C.byref(n)) == 0
    nodes = (C.c_void_p * n.value)()
    assert rt.cudaGraphGetNodes(raw, nodes, C.byref(n)) == 0
    kernels = cleared = others = 0
    for node in nodes:
        kind, m = C.c_int(), Memset()
        assert rt.cudaGraphNodeGetType(C.c_void_p(node), C.byref(kind)) == 0
        if kind.value == 0:
            kernels += 1
        elif kind.value == 2:
            assert rt.cudaGraphMemsetNodeGetParams(C.c_void_p(node), C.byref(m)) == 0
            cleared += m.element * m.width * m.height
        else:
            others += 1
    return kernels, cleared, others


def test_captured_calls_do_nothing_but_their_kernels():
    """One kernel a call, and one clear of the counters for all calls of an operator."""
    import torch
    from ktir_cpu_b200 import check_status, kv_append, paged_decode, prompt_attention
    q, kc, vc, pages, lengths = _decode_inputs("bf16", [300, 77, 5], 8, 2, 128, 16, seed=57)
    k, v = kc[0, :3].clone(), vc[0, :3].clone()
    p = _prompt_inputs("bf16", [64, 9], [3000, 9], 8, 2, 128, seed=57)
    slots = torch.tensor([-1, -1, -1], dtype=torch.int32, device="cuda")
    want, want2 = paged_decode(q, kc, vc, pages, lengths), prompt_attention(*p[:4], kv_offsets=p[4])
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        for _ in range(6):
            turned = kv_append(k, v, kc, vc, slots, q=q)
            got = paged_decode(turned, kc, vc, pages, lengths)
            got2 = prompt_attention(*p[:4], kv_offsets=p[4])
    kernels, cleared, others = _nodes(graph)
    assert (kernels, others) == (18, 0)
    assert cleared == 3 * 2 * 4 + 160 * 4            # sequences x head tiles; row tiles that share keys
    graph.instantiate()
    for _ in range(3):
        graph.replay()
        assert torch.equal(got, want) and torch.equal(got2, want2)
    check_status()


@pytest.mark.parametrize("order", [1, -1])
def test_captured_calls_of_many_sizes(order):
    """Calls that split sequences and row tiles and calls that do not, of rising and
    falling sizes, in one graph and on two streams of it: what a graph's later calls
    allocate may lie where its earlier ones had their workspace."""
    import torch
    from ktir_cpu_b200 import check_status, paged_decode, prompt_attention
    decodes = [_decode_inputs("bf16", n, 8, 2, 128, 16, seed=58)
               for n in ([5000], [3000, 17, 400], [2000] * 40, [900] * 200, [0, 6000])][::order]
    prompts = [_prompt_inputs("bf16", new, keys, 8, 2, 128, seed=59)
               for new, keys in (([64], [8192]), ([5], [900]), ([30] * 60, [30] * 60), ([16] * 4, [5000] * 4))][::order]
    attend = lambda p: prompt_attention(*p[:4], kv_offsets=p[4])  # noqa: E731
    want = [paged_decode(*x) for x in decodes], [attend(p) for p in prompts]
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    for _ in range(2):                               # the second capture after the first has been replayed
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            main = torch.cuda.current_stream()
            side.wait_stream(main)
            got = [], []
            for i in range(5):
                got[0].append(paged_decode(*decodes[i]))
                got[1].append(attend(prompts[i % 4]))
                with torch.cuda.stream(side):
                    got[0].append(paged_decode(*decodes[4 - i]))
                    got[1].append(attend(prompts[3 - i % 4]))
            main.wait_stream(side)
        for _ in range(20):
            for t in got[0] + got[1]:
                t.zero_()
            graph.replay()
            eager = paged_decode(*decodes[0]), attend(prompts[0])
            for i in range(5):
                assert torch.equal(got[0][2 * i], want[0][i]) and torch.equal(got[0][2 * i + 1], want[0][4 - i])
                assert torch.equal(got[1][2 * i], want[1][i % 4]) and torch.equal(got[1][2 * i + 1], want[1][3 - i % 4])
            assert torch.equal(eager[0], want[0][0]) and torch.equal(eager[1], want[1][0])
    check_status()


def test_what_is_no_tensor_is_refused():
    import torch
    from ktir_cpu_b200 import kv_append, paged_decode, prompt_attention
    q, kc, vc, pages, lengths = _decode_inputs("bf16", [40, 20], 4, 2, 64, 16, seed=60)
    k = kc[0, :2]
    off = torch.tensor([0, 2], dtype=torch.int32, device="cuda")
    appends = [k, k, kc, vc, off, q, off, torch.zeros(8, 64, device="cuda")]
    append = lambda *a: kv_append(*a[:5], q=a[5], positions=a[6], table=a[7], q_out=a[8])  # noqa: E731
    for call, args in [(append, appends + [torch.empty_like(q)]), (lambda *a: paged_decode(*a[:5], out=a[5]),
                                                                 [q, kc, vc, pages, lengths, torch.empty_like(q)]),
                       (lambda *a: prompt_attention(*a[:5], out=a[5]), [k, k, k, off, off, torch.empty_like(k)])]:
        call(*args)
        for at in range(len(args)):
            for wrong in (3, "k", [1, 2]):
                with pytest.raises(ValueError, match="must be"):
                    call(*args[:at], wrong, *args[at + 1:])


# -- reach of what is not finite, calls without a workspace, many sequences ----------------

@pytest.mark.parametrize("n,heads,kv_heads,dim", [(256, 4, 1, 128), (256, 2, 2, 64), (3000, 8, 8, 128), (3000, 16, 4, 64)])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_prompt_reach_of_infinite_values(n, heads, kv_heads, dim, bad):
    """A value row that is not finite reaches no row tile whose last block of keys ends
    before it, and no other kv head."""
    import torch
    from ktir_cpu_b200 import check_status, prompt_attention
    q, k, v, offsets, _ = _prompt_inputs("bf16", [n], [n], heads, kv_heads, dim, seed=61)
    clean = prompt_attention(q, k, v, offsets)
    group = heads // kv_heads
    tile, block = 128 // group, 80 if dim == 128 else 128
    for at in (n // 3, n // 2 + 17, n - 1):
        v2 = v.clone()
        v2[at, 0] = bad
        got = prompt_attention(q, k, v2, offsets)
        first = next(t for t in range(0, n, tile) if -(-min(n, t + tile) // block) * block > at)
        assert at - first < tile + block
        assert torch.equal(got[:first], clean[:first]) and torch.equal(got[:, group:], clean[:, group:])
        assert not torch.isfinite(got[at:, :group]).any()
    check_status()


@pytest.mark.parametrize("new,keys,dim", [([64], [8192], 128), ([16] * 4, [5000] * 4, 64), ([300], [300], 64)])
def test_prompt_without_a_workspace(new, keys, dim):
    """The C entry with no workspace: the keys of few queries are not shared out."""
    import ctypes
    import torch
    from ktir_cpu_b200 import runtime as R
    q, k, v, offsets, kv_offsets = _prompt_inputs("bf16", new, keys, 8, 2, dim, seed=62)
    out, lse = torch.empty_like(q), torch.empty(q.shape[:2], device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    d = R.KtirPromptDesc()
    for name, t in (("q", q), ("k", k), ("v", v), ("out", out), ("lse", lse), ("offsets", offsets),
                    ("kv_offsets", kv_offsets), ("status", status)):
        setattr(d, name, t.data_ptr())
    for name, t in (("q_stride", q), ("k_stride", k), ("v_stride", v), ("out_stride", out)):
        getattr(d, name)[0], getattr(d, name)[1] = t.stride(0), t.stride(1)
    d.batch, d.tokens, d.kv_tokens = len(new), q.shape[0], k.shape[0]
    d.heads, d.kv_heads, d.dim, d.dtype, d.scale, d.causal = 8, 2, dim, R.BF16, dim ** -0.5, 1
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    assert R.load_library().ktir_prompt_attention(ctypes.byref(d), stream) == 0
    torch.cuda.synchronize()
    assert not int(status)
    _check_prompt("bf16", q, k, v, offsets, kv_offsets, True, dim ** -0.5, out, lse)


def test_prompt_thousands_of_sequences():
    from ktir_cpu_b200 import check_status, prompt_attention
    rng = random.Random(9)
    new = [rng.choice([0, 0, 1, 1, 2, 9, 33, 150]) for _ in range(3000)]
    x = _prompt_inputs("f16", new, new, 1, 1, 64, seed=63)
    out, lse = prompt_attention(*x[:4], return_lse=True)
    check_status()
    _check_prompt("f16", *x, True, 0.125, out, lse)


def test_prompt_time_grows_with_the_sequences():
    """Four times the sequences of few tokens take about four times as long, not sixteen;
    and they are right at the batch's end."""
    import torch
    from ktir_cpu_b200 import check_status, prompt_attention

    def timed(batch):
        gen = _gen(batch)
        new = torch.randint(1, 40, (batch,), generator=gen, device="cuda")
        offsets = torch.cat([torch.zeros(1, dtype=torch.int64, device="cuda"), new.cumsum(0)]).int()
        n = int(offsets[-1])
        q, k, v = (_randn(gen, "bf16", n, h, 64) for h in (4, 2, 2))
        prompt_attention(q, k, v, offsets)
        best = math.inf
        for _ in range(5):
            a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            a.record()
            out, lse = prompt_attention(q, k, v, offsets, return_lse=True)
            b.record()
            torch.cuda.synchronize()
            best = min(best, a.elapsed_time(b))
        for at in (0, batch // 2, batch - 200):
            ends = offsets[at:at + 201]
            lo, hi = int(ends[0]), int(ends[-1])
            _check_prompt("bf16", q[lo:hi], k[lo:hi], v[lo:hi], ends - lo, ends - lo, True, 0.125, out[lo:hi], lse[lo:hi])
        return best

    few, many = timed(5000), timed(20000)
    check_status()
    assert many < 8 * few, (few, many)


@pytest.mark.parametrize("causal", [True, False])
def test_prompt_many_weights_over_many_sequences(causal):
    """More sequences than a block keeps the lengths of, of many key counts, some beyond
    the table of weights: every tile is found once."""
    import torch
    from ktir_cpu_b200 import check_status, prompt_attention
    rng = random.Random(11)
    for longest in (600, 45000):
        new = [rng.choice([0, 1, 3, 40, 130, 300]) for _ in range(400)]
        keys = [n + rng.choice([0, 0, 5, 700]) if n else 0 for n in new]
        new[333], keys[333] = 200, longest
        q, k, v, offsets, kv_offsets = _prompt_inputs("bf16", new, keys, 2, 1, 128, seed=64)
        out, lse = prompt_attention(q, k, v, offsets, kv_offsets=kv_offsets, causal=causal, return_lse=True)
        check_status()
        _check_prompt("bf16", q, k, v, offsets, kv_offsets, causal, 128 ** -0.5, out, lse)
