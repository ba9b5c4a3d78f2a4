"""The serving operators without a GPU: descriptor layouts, refusals."""

import ctypes as C
import os
import shutil
import subprocess

import pytest

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "ktir_b200.h")
STRUCTS = ["KtirKvAppendDesc", "KtirPagedDecodeDesc", "KtirPromptDesc"]


@pytest.mark.skipif(shutil.which("gcc") is None, reason="needs gcc")
def test_layouts(tmp_path):
    from ktir_cpu_b200 import runtime as R
    lines = []
    for s in STRUCTS:
        lines.append(f'printf("%zu\\n", sizeof({s}));')
        lines += [f'printf("%zu\\n", offsetof({s}, {f[0]}));' for f in getattr(R, s)._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "ktir_b200.h"\nint main(void){\n'
                   + "\n".join(lines) + "\nreturn 0;}\n")
    exe = tmp_path / "layout"
    subprocess.check_call(["gcc", "-I", os.path.dirname(HEADER), str(src), "-o", str(exe)])
    got = list(map(int, subprocess.check_output([str(exe)]).split()))
    want = []
    for s in STRUCTS:
        t = getattr(R, s)
        want += [C.sizeof(t)] + [getattr(t, f[0]).offset for f in t._fields_]
    assert got == want


def _decode_desc(**change):
    from ktir_cpu_b200 import runtime as R
    d = R.KtirPagedDecodeDesc()
    for f in ("q", "k_cache", "v_cache", "out", "pages", "lengths", "workspace", "status"):
        setattr(d, f, 1 << 20)
    d.workspace_bytes = 1 << 40
    d.batch, d.max_pages, d.page_row, d.num_pages, d.page_size = 2, 4, 4, 8, 16
    d.heads, d.kv_heads, d.dim, d.dtype, d.scale = 8, 2, 128, R.BF16, 0.1
    for name, n in (("q_stride", 2), ("out_stride", 2), ("kc_stride", 3), ("vc_stride", 3)):
        for i in range(n):
            getattr(d, name)[i] = 128
    for key, value in change.items():
        setattr(d, key, value)
    return d


def _prompt_desc(**change):
    from ktir_cpu_b200 import runtime as R
    d = R.KtirPromptDesc()
    for f in ("q", "k", "v", "out", "offsets", "kv_offsets", "status"):
        setattr(d, f, 1 << 20)
    d.batch, d.tokens, d.kv_tokens = 2, 10, 10
    d.heads, d.kv_heads, d.dim, d.dtype, d.scale = 8, 2, 128, R.F16, 0.1
    for name in ("q_stride", "k_stride", "v_stride", "out_stride"):
        getattr(d, name)[0], getattr(d, name)[1] = 1024, 128
    for key, value in change.items():
        setattr(d, key, value)
    return d


def _append_desc(**change):
    from ktir_cpu_b200 import runtime as R
    d = R.KtirKvAppendDesc()
    for f in ("k", "v", "k_cache", "v_cache", "slots", "positions", "table", "status"):
        setattr(d, f, 1 << 20)
    d.tokens, d.num_pages, d.page_size, d.table_rows, d.table_stride = 3, 4, 16, 100, 128
    d.heads, d.kv_heads, d.dim, d.rot, d.dtype = 8, 2, 128, 128, R.BF16
    for name, n in (("k_stride", 2), ("v_stride", 2), ("kc_stride", 3), ("vc_stride", 3)):
        for i in range(n):
            getattr(d, name)[i] = 128
    for key, value in change.items():
        setattr(d, key, value)
    return d


ARG, UNSUPPORTED = -1, -3


@pytest.mark.parametrize("change,code", [
    (dict(q=0), ARG), (dict(workspace=0), ARG), (dict(workspace_bytes=0), ARG), (dict(kv_heads=3), ARG),
    (dict(page_size=0), ARG), (dict(max_pages=0), ARG), (dict(batch=-1), ARG), (dict(dim=96), UNSUPPORTED),
    (dict(dtype=1), UNSUPPORTED), (dict(scale=0.0), UNSUPPORTED), (dict(scale=float("inf")), UNSUPPORTED),
    (dict(q=(1 << 20) + 2), UNSUPPORTED), (dict(v_cache=(1 << 20) + 8), UNSUPPORTED),
])
def test_decode_refusals(change, code):
    from ktir_cpu_b200 import runtime as R
    lib = R.load_library()
    assert lib.ktir_paged_decode(C.byref(_decode_desc(**change)), None) == code
    assert lib.ktir_last_error().startswith(b"ktir_paged_decode")
    bent = _decode_desc()
    bent.kc_stride[1] = 100
    assert lib.ktir_paged_decode(C.byref(bent), None) == UNSUPPORTED
    assert lib.ktir_paged_decode(None, None) == ARG
    assert lib.ktir_paged_decode(C.byref(_decode_desc(batch=0)), None) == 0


@pytest.mark.parametrize("change,code", [
    (dict(k=0), ARG), (dict(offsets=0), ARG), (dict(kv_heads=3), ARG), (dict(batch=0), ARG),
    (dict(tokens=-1), ARG), (dict(kv_tokens=1 << 31), ARG), (dict(dim=80), UNSUPPORTED),
    (dict(dtype=1), UNSUPPORTED), (dict(heads=258), UNSUPPORTED), (dict(scale=-0.5), UNSUPPORTED),
    (dict(out=(1 << 20) + 4), UNSUPPORTED),
])
def test_prompt_refusals(change, code):
    from ktir_cpu_b200 import runtime as R
    lib = R.load_library()
    assert lib.ktir_prompt_attention(C.byref(_prompt_desc(**change)), None) == code
    assert lib.ktir_last_error().startswith(b"ktir_prompt_attention")
    bent = _prompt_desc()
    bent.v_stride[0] = 1028
    assert lib.ktir_prompt_attention(C.byref(bent), None) == UNSUPPORTED
    assert lib.ktir_prompt_attention(C.byref(_prompt_desc(tokens=0)), None) == 0


@pytest.mark.parametrize("change,code", [
    (dict(slots=0), ARG), (dict(positions=0), ARG), (dict(q=1 << 20), ARG), (dict(table_rows=0), ARG),
    (dict(page_size=0), ARG), (dict(dim=264), UNSUPPORTED), (dict(rot=24), UNSUPPORTED),
    (dict(rot=256), UNSUPPORTED), (dict(dtype=2), UNSUPPORTED), (dict(k=(1 << 20) + 2), UNSUPPORTED),
])
def test_append_refusals(change, code):
    from ktir_cpu_b200 import runtime as R
    lib = R.load_library()
    assert lib.ktir_kv_append(C.byref(_append_desc(**change)), None) == code
    assert lib.ktir_last_error().startswith(b"ktir_kv_append")
    bent = _append_desc()
    bent.k_stride[0] = 132
    assert lib.ktir_kv_append(C.byref(bent), None) == UNSUPPORTED
    assert lib.ktir_kv_append(C.byref(_append_desc(tokens=0)), None) == 0


def test_cpu_tensors_are_refused():
    torch = pytest.importorskip("torch")
    from ktir_cpu_b200 import kv_append, paged_decode, prompt_attention
    x = torch.zeros(2, 4, 64, dtype=torch.bfloat16)
    c = torch.zeros(3, 8, 2, 64, dtype=torch.bfloat16)
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        paged_decode(x, c, c, i[:, None], i)
    with pytest.raises(ValueError, match="CUDA"):
        prompt_attention(x, x, x, i)
    with pytest.raises(ValueError, match="CUDA"):
        kv_append(x, x, c, c, i)


class _FakeBinding:
    """The binding's status word of one device, in host memory."""

    def __init__(self, value):
        import torch
        self.word = torch.tensor([value], dtype=torch.int32)
        self.forgotten = []

    def forget(self, dev):
        self.forgotten.append(dev)

    def status(self, dev):
        return self.word


@pytest.mark.parametrize("bits,kind,text", [
    (0, None, None), ("bad", IndexError, "out of range"), ("timeout", RuntimeError, "timed out"),
    ("both", RuntimeError, "timed out.*out of range"),
])
def test_check_status_reports_every_bit(monkeypatch, bits, kind, text):
    torch = pytest.importorskip("torch")
    from ktir_cpu_b200 import runtime as R
    from ktir_cpu_b200 import serving
    value = {0: 0, "bad": R.STATUS_BAD_INDEX, "timeout": R.STATUS_TIMEOUT,
             "both": R.STATUS_BAD_INDEX | R.STATUS_TIMEOUT}[bits]
    fake = _FakeBinding(value)
    monkeypatch.setattr(serving, "_EXT", fake)
    monkeypatch.setattr(torch.cuda, "synchronize", lambda dev=None: None)
    if kind is None:
        serving.check_status(0)
    else:
        with pytest.raises(kind, match=text):
            serving.check_status(0)
    assert int(fake.word) == 0
    serving.check_status(0)


@pytest.mark.parametrize("timeout", [False, True])
def test_workspaces_are_given_up_after_a_timeout(monkeypatch, timeout):
    """A split call that was given up leaves counters that a later call would take for its own."""
    torch = pytest.importorskip("torch")
    from ktir_cpu_b200 import runtime as R
    from ktir_cpu_b200 import serving
    fake = _FakeBinding(R.STATUS_TIMEOUT if timeout else R.STATUS_BAD_INDEX)
    monkeypatch.setattr(serving, "_EXT", fake)
    monkeypatch.setattr(torch.cuda, "synchronize", lambda dev=None: None)
    with pytest.raises(RuntimeError if timeout else IndexError):
        serving.check_status(3)
    assert fake.forgotten == ([3] if timeout else [])


def test_written_tensors_do_not_share_memory():
    """Outputs and caches with an expanded axis are refused (many tokens, one place);
    one entry along it needs no stride."""
    from ktir_cpu_b200 import runtime as R
    lib = R.load_library()
    for call, make, names in [
        (lib.ktir_kv_append, lambda **c: _append_desc(q=1 << 20, q_out=1 << 20, **c), ("qo_stride", "kc_stride", "vc_stride")),
        (lib.ktir_paged_decode, _decode_desc, ("out_stride",)),
        (lib.ktir_prompt_attention, _prompt_desc, ("out_stride",)),
    ]:
        for name in names:
            d = make()
            for other in ("q_stride", "qo_stride"):
                if hasattr(d, other):
                    getattr(d, other)[0], getattr(d, other)[1] = 1024, 128
            for axis in range(len(getattr(d, name))):
                was, getattr(d, name)[axis] = getattr(d, name)[axis], 0
                assert call(C.byref(d), None) == ARG, (name, axis)
                assert b"share memory" in lib.ktir_last_error()
                getattr(d, name)[axis] = was


@pytest.mark.parametrize("wrong", [None, 3, [1.0, 2.0]])
def test_what_is_no_tensor_is_refused(wrong):
    torch = pytest.importorskip("torch")
    from ktir_cpu_b200 import kv_append, paged_decode, prompt_attention
    x = torch.zeros(2, 4, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="k must be a tensor"):
        kv_append(wrong, x, x, x, x)
    with pytest.raises(ValueError, match="q must be a tensor"):
        paged_decode(wrong, x, x, x, x)
    with pytest.raises(ValueError, match="q must be a tensor"):
        prompt_attention(wrong, x, x, x)


def test_prompt_batch_limit():
    """The kernel looks at every sequence in every block: a call has a bound on them."""
    from ktir_cpu_b200 import runtime as R
    lib = R.load_library()
    assert lib.ktir_prompt_attention(C.byref(_prompt_desc(batch=(1 << 20) + 1)), None) == UNSUPPORTED
    assert b"2^20" in lib.ktir_last_error()
