"""The C ABI of include/afa_sm100_ops.h without a GPU: exported symbols, the
ctypes mirrors against a C program, argument errors before any CUDA call."""

import ctypes
import re
import subprocess
from pathlib import Path

import pytest

from ampere_flash_attention_from_scratch_b200 import _abi

ROOT = Path(__file__).resolve().parents[1]
HEADER = ROOT / "include" / "afa_sm100_ops.h"
STRUCTS = {"AfaRotaryArgs": _abi.AfaRotaryArgs, "AfaCache4": _abi.AfaCache4, "AfaCache4FwdArgs": _abi.AfaCache4FwdArgs}


def test_every_declared_symbol_is_exported():
    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)
    names = set(re.findall(r"^\s*(?:int|int32_t|int64_t)\s+(afa_\w+)\s*\(", text, flags=re.M))
    assert names == set(_abi.EXPORTED_OPS_SYMBOLS)
    lib = _abi.load()
    assert all(hasattr(lib, n) for n in names)
    assert lib.afa_sm100_ops_version() == 100


@pytest.mark.parametrize("name", STRUCTS)
def test_struct_layout_matches_c(name, tmp_path):
    cls = STRUCTS[name]
    fields = [f for f, _ in cls._fields_]
    src = tmp_path / "layout.c"
    body = "\n".join(f'  printf("{f} %zu\\n", offsetof({name}, {f}));' for f in fields)
    src.write_text(f'#include <stdio.h>\n#include <stddef.h>\n#include "afa_sm100_ops.h"\nint main(void) {{\n'
                   f'  printf("sizeof %zu\\n", sizeof({name}));\n{body}\n  return 0;\n}}\n')
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c99", f"-I{ROOT / 'include'}", str(src), "-o", str(exe)], check=True)
    out = dict(x.split() for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines())
    assert int(out["sizeof"]) == ctypes.sizeof(cls)
    for f in fields:
        assert int(out[f]) == getattr(cls, f).offset, f


def _set(struct, over):
    for k, v in over.items():
        if isinstance(v, (list, tuple)):
            getattr(struct, k)[:] = v
        else:
            setattr(struct, k, v)
    return struct


def rotary_args(**over):
    a = _abi.AfaRotaryArgs()
    a.q = a.k = a.q_out = a.k_out = a.positions = a.inv_freq = 0x100000
    for n in ("q_strides", "q_out_strides", "k_strides", "k_out_strides"):
        getattr(a, n)[:] = [16 * 4 * 128, 4 * 128, 128]
    a.pos_strides[:] = [32, 16, 1]
    a.sections[:] = [16, 24, 24, 0, 0, 0, 0, 0]
    a.n_axes, a.pos_type = 3, _abi.AFA_POS_INT64
    a.batch, a.seq_len, a.n_heads, a.n_k_heads, a.head_dim, a.rot_dim = 2, 16, 4, 4, 128, 128
    a.dtype = _abi.AFA_DTYPE_BF16
    return _set(a, over)


@pytest.mark.parametrize("over,code", [
    (dict(dtype=6), _abi.AFA_ERR_UNSUPPORTED_DTYPE),
    (dict(head_dim=120), _abi.AFA_ERR_NO_KERNEL),
    (dict(head_dim=528), _abi.AFA_ERR_NO_KERNEL),
    (dict(rot_dim=144), _abi.AFA_ERR_NO_KERNEL),
    (dict(rot_dim=24), _abi.AFA_ERR_NO_KERNEL),
    (dict(rot_dim=0), _abi.AFA_ERR_NO_KERNEL),
    (dict(q=None), _abi.AFA_ERR_INVALID_ARGUMENT),
    (dict(k_out=None), _abi.AFA_ERR_INVALID_ARGUMENT),
    (dict(positions=None), _abi.AFA_ERR_INVALID_ARGUMENT),
    (dict(inv_freq=None), _abi.AFA_ERR_INVALID_ARGUMENT),
    (dict(batch=0), _abi.AFA_ERR_INVALID_ARGUMENT),
    (dict(seq_len=-1), _abi.AFA_ERR_INVALID_ARGUMENT),
    (dict(n_k_heads=0), _abi.AFA_ERR_INVALID_ARGUMENT),
    (dict(n_axes=0), _abi.AFA_ERR_INVALID_ARGUMENT),
    (dict(n_axes=9), _abi.AFA_ERR_INVALID_ARGUMENT),
    (dict(pos_type=3), _abi.AFA_ERR_INVALID_ARGUMENT),
    (dict(interleaved=2), _abi.AFA_ERR_INVALID_ARGUMENT),
    (dict(inverse=-1), _abi.AFA_ERR_INVALID_ARGUMENT),
    (dict(sections=[16, 24, 23, 0, 0, 0, 0, 0]), _abi.AFA_ERR_INVALID_ARGUMENT),
    (dict(sections=[-16, 40, 40, 0, 0, 0, 0, 0]), _abi.AFA_ERR_INVALID_ARGUMENT),
    (dict(q=0x100008), _abi.AFA_ERR_MISALIGNED),
    (dict(positions=0x100004), _abi.AFA_ERR_MISALIGNED),
    (dict(q_strides=[8192, 512, 124]), _abi.AFA_ERR_MISALIGNED),
    (dict(q_out_strides=[0, 512, 128]), _abi.AFA_ERR_MISALIGNED),  # outputs may not repeat
    (dict(batch=1 << 20, seq_len=1 << 20), _abi.AFA_ERR_TOO_LARGE),
])
def test_rotary_argument_errors(over, code):
    assert _abi.load().afa_rotary_sm100(ctypes.byref(rotary_args(**over)), None) == code


def test_rotary_null_and_without_k():
    lib = _abi.load()
    assert lib.afa_rotary_sm100(None, None) == _abi.AFA_ERR_INVALID_ARGUMENT
    early = {_abi.AFA_ERR_INVALID_ARGUMENT, _abi.AFA_ERR_MISALIGNED, _abi.AFA_ERR_NO_KERNEL}
    # valid arguments get past the checks; on a machine without a GPU the device is what is missing
    for a in (rotary_args(k=None, k_out=None, n_k_heads=0), rotary_args(q_strides=[0, 0, 128])):
        if lib.afa_fwd_sm100(None, None) and not _gpu():
            assert lib.afa_rotary_sm100(ctypes.byref(a), None) not in early


def _gpu():
    import torch

    return torch.cuda.is_available()


def cache(**over):
    c = _abi.AfaCache4()
    c.cache = c.page_table = c.kv_lens = 0x100000
    c.page_stride = 4 * 2 * 64 * 72
    c.table_stride = 16
    c.n_pages, c.page_size, c.max_pages, c.batch, c.n_kv_heads, c.head_dim = 100, 64, 16, 3, 4, 128
    c.dtype = _abi.AFA_DTYPE_FP16
    return _set(c, over)


CACHE_ERRORS = [
    (dict(dtype=1), _abi.AFA_ERR_UNSUPPORTED_DTYPE),
    (dict(head_dim=96), _abi.AFA_ERR_NO_KERNEL),
    (dict(cache=None), _abi.AFA_ERR_INVALID_ARGUMENT),
    (dict(page_table=None), _abi.AFA_ERR_INVALID_ARGUMENT),
    (dict(kv_lens=None), _abi.AFA_ERR_INVALID_ARGUMENT),
    (dict(n_pages=0), _abi.AFA_ERR_INVALID_ARGUMENT),
    (dict(max_pages=0), _abi.AFA_ERR_INVALID_ARGUMENT),
    (dict(batch=-3), _abi.AFA_ERR_INVALID_ARGUMENT),
    (dict(n_kv_heads=0), _abi.AFA_ERR_INVALID_ARGUMENT),
    (dict(page_size=8), _abi.AFA_ERR_INVALID_ARGUMENT),
    (dict(page_size=48), _abi.AFA_ERR_INVALID_ARGUMENT),
    (dict(page_size=512), _abi.AFA_ERR_INVALID_ARGUMENT),
    (dict(page_stride=0), _abi.AFA_ERR_INVALID_ARGUMENT),
    (dict(page_stride=4 * 2 * 64 * 72 - 16), _abi.AFA_ERR_INVALID_ARGUMENT),
    (dict(table_stride=-16), _abi.AFA_ERR_INVALID_ARGUMENT),
    (dict(cache=0x100008), _abi.AFA_ERR_MISALIGNED),
    (dict(page_stride=4 * 2 * 64 * 72 + 8), _abi.AFA_ERR_MISALIGNED),
    (dict(page_table=0x100002), _abi.AFA_ERR_MISALIGNED),
    (dict(kv_lens=0x100001), _abi.AFA_ERR_MISALIGNED),
    (dict(new_lens=0x100002), _abi.AFA_ERR_MISALIGNED),
    (dict(max_pages=1 << 26), _abi.AFA_ERR_TOO_LARGE),
]


def _strides(*s):
    return (ctypes.c_int64 * 3)(*s)


GOOD = (16 * 512, 512, 128)


def call(which, c, k=0x100000, v=0x100000, ks=GOOD, vs=GOOD, n=16):
    fn = getattr(_abi.load(), f"afa_cache4_{which}_sm100")
    return fn(ctypes.byref(c) if c else None, k, v, _strides(*ks), _strides(*vs), n, None)


@pytest.mark.parametrize("over,code", CACHE_ERRORS)
def test_cache_argument_errors(over, code):
    c = cache(**over)
    lib = _abi.load()
    assert call("write", c) == code
    assert call("read", c) == code
    assert lib.afa_cache4_fwd_workspace(ctypes.byref(c), 1, 8) == -code
    assert lib.afa_cache4_fwd_sm100(ctypes.byref(c), ctypes.byref(fwd_args()), None) == code


@pytest.mark.parametrize("over,code", [
    (dict(k=None), _abi.AFA_ERR_INVALID_ARGUMENT),
    (dict(v=None), _abi.AFA_ERR_INVALID_ARGUMENT),
    (dict(n=0), _abi.AFA_ERR_INVALID_ARGUMENT),
    (dict(k=0x100004), _abi.AFA_ERR_MISALIGNED),
    (dict(vs=(8192, 516, 128)), _abi.AFA_ERR_MISALIGNED),
])
@pytest.mark.parametrize("which", ["write", "read"])
def test_move_argument_errors(which, over, code):
    assert call(which, cache(), **over) == code


def test_only_the_writer_takes_repeated_rows():
    assert call("read", cache(), ks=(0, 512, 128)) == _abi.AFA_ERR_MISALIGNED
    if not _gpu():
        assert call("write", cache(), ks=(0, 512, 128)) != _abi.AFA_ERR_MISALIGNED
    assert call("write", None) == call("read", None) == _abi.AFA_ERR_INVALID_ARGUMENT


def fwd_args(**over):
    a = _abi.AfaCache4FwdArgs()
    a.q = a.o = a.workspace = 0x100000
    a.q_strides[:] = a.o_strides[:] = [8 * 128, 8 * 128, 128]
    a.workspace_bytes = 1 << 30
    a.seq_len, a.n_heads = 1, 8
    return _set(a, over)


@pytest.mark.parametrize("over,code", [
    (dict(q=None), _abi.AFA_ERR_INVALID_ARGUMENT),
    (dict(o=None), _abi.AFA_ERR_INVALID_ARGUMENT),
    (dict(workspace=None), _abi.AFA_ERR_INVALID_ARGUMENT),
    (dict(seq_len=0), _abi.AFA_ERR_INVALID_ARGUMENT),
    (dict(n_heads=0), _abi.AFA_ERR_INVALID_ARGUMENT),
    (dict(n_heads=6), _abi.AFA_ERR_INVALID_ARGUMENT),  # not a multiple of 4 key/value heads
    (dict(causal=2), _abi.AFA_ERR_INVALID_ARGUMENT),
    (dict(scale=float("nan")), _abi.AFA_ERR_INVALID_ARGUMENT),
    (dict(scale=3e38), _abi.AFA_ERR_INVALID_ARGUMENT),
    (dict(q=0x100008), _abi.AFA_ERR_MISALIGNED),
    (dict(workspace=0x100008), _abi.AFA_ERR_MISALIGNED),
    (dict(lse=0x100002), _abi.AFA_ERR_MISALIGNED),
    (dict(o_strides=[1024, 1024, 0]), _abi.AFA_ERR_MISALIGNED),
    (dict(seq_len=1 << 30), _abi.AFA_ERR_TOO_LARGE),
])
def test_fwd_argument_errors(over, code):
    a = fwd_args(**over)
    assert _abi.load().afa_cache4_fwd_sm100(ctypes.byref(cache()), ctypes.byref(a), None) == code


def test_fwd_null_and_row_bytes():
    lib = _abi.load()
    assert lib.afa_cache4_fwd_sm100(ctypes.byref(cache()), None, None) == _abi.AFA_ERR_INVALID_ARGUMENT
    assert lib.afa_cache4_fwd_sm100(None, ctypes.byref(fwd_args()), None) == _abi.AFA_ERR_INVALID_ARGUMENT
    assert [lib.afa_cache4_row_bytes(d) for d in (64, 128, 96, 0)] == [36, 72, -1, -1]
    assert b"page_table" in lib.afa_status_string(_abi.AFA_DEV_BAD_PAGE)
    assert b"kv_lens" in lib.afa_status_string(_abi.AFA_DEV_BAD_LENGTH)
