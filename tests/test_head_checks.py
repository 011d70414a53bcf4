"""top_logits and sample_logits without a GPU: what the Python layer and the C ABI refuse, before any device is touched."""
import ctypes

import pytest
import torch

from linear_cross_entropy_loss_b200 import _native, sample_logits, top_logits


@pytest.fixture(scope="module")
def lib():
    return _native.load()


@pytest.mark.parametrize("kw", [dict(k=0), dict(k=-1), dict(k=9), dict(k=3, temperature=0.0), dict(k=3, temperature=-1.0),
                                dict(k=3, temperature=float("nan"))])
def test_top_logits_refuses(kw):
    with pytest.raises(AssertionError):
        top_logits(torch.zeros(2, 8), **kw)


def test_top_logits_refuses_long_lists_and_other_types():
    with pytest.raises(AssertionError):
        top_logits(torch.zeros(2, 5000), 1025)
    with pytest.raises(AssertionError):
        top_logits(torch.zeros(2, 8, dtype=torch.float64), 2)
    with pytest.raises(AssertionError):
        top_logits(torch.zeros(2, 0), 1)


@pytest.mark.parametrize("kw", [
    dict(temperature=-0.1), dict(temperature=float("nan")), dict(top_k=-1), dict(top_p=0.0), dict(top_p=1.1),
    dict(top_p=float("nan")), dict(min_p=-0.1), dict(min_p=1.5), dict(temperature=torch.ones(3)),
    dict(top_k=torch.ones(2)), dict(top_p=torch.ones(5)),
])
def test_sample_logits_refuses(kw):
    with pytest.raises(AssertionError):
        sample_logits(torch.zeros(2, 8), torch.zeros(2), **kw)


def test_sample_logits_refuses_other_random_numbers():
    with pytest.raises(AssertionError):
        sample_logits(torch.zeros(2, 8), torch.zeros(3))
    with pytest.raises(AssertionError):
        sample_logits(torch.zeros(2, 8), torch.zeros(2, dtype=torch.float16))


def test_there_is_no_cpu_fallback():
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        top_logits(torch.zeros(2, 8), 2)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        sample_logits(torch.zeros(2, 8), torch.zeros(2))


@pytest.mark.parametrize("change,code", [
    (dict(dtype=3), -1), (dict(dtype=-1), -1), (dict(logits=None), -1), (dict(ld=-1), -1), (dict(rows=-1), -1),
    (dict(vocab=0), -1), (dict(k=0), -1), (dict(t=0.0), -1), (dict(t=float("nan")), -1), (dict(values=None), -1),
    (dict(indices=None), -1), (dict(lse=None), -1), (dict(k=101), -8), (dict(vocab=4000, k=1025), -8),
    (dict(vocab=1 << 31), -8), (dict(rows=1 << 31), -8), (dict(logits=17), -3), (dict(dtype=2, logits=18), -3),
])
def test_top_logits_abi_refuses(lib, change, code):
    a = dict(dtype=1, logits=16, ld=100, rows=4, vocab=100, k=8, t=1.0, values=16, indices=16, lse=16)
    a.update(change)
    assert lib.lce_top_logits(a["dtype"], a["logits"], a["ld"], a["rows"], a["vocab"], a["k"], a["t"], a["values"],
                              a["indices"], a["lse"], None) == code


@pytest.mark.parametrize("change", [dict(ld=-1), dict(rows=-1), dict(vocab=0), dict(dtype=9)])
def test_sample_logits_abi_refuses_shapes(lib, change):
    a = dict(dtype=1, logits=16, ld=100, rows=4, vocab=100)
    a.update(change)
    s = sampling()
    assert lib.lce_sample_logits(a["dtype"], a["logits"], a["ld"], a["rows"], a["vocab"], ctypes.byref(s), 16, 16, None) == -1


def sampling(**kw):
    base = dict(u=16, temperature_all=1.0, top_p_all=1.0, min_p_all=0.0, top_k_all=0, u_dtype=_native.DTYPE_F32)
    base.update(kw)
    return _native.Sampling(**base)


@pytest.mark.parametrize("kw", [
    dict(u=None), dict(u_dtype=0), dict(u_dtype=4), dict(temperature_all=-1.0), dict(temperature_all=float("nan")),
    dict(top_p_all=0.0), dict(top_p_all=1.5), dict(top_p_all=float("nan")), dict(min_p_all=-0.5), dict(min_p_all=2.0),
    dict(min_p_all=float("nan")), dict(top_k_all=-3),
])
def test_sample_logits_abi_refuses(lib, kw):
    s = sampling(**kw)
    assert lib.lce_sample_logits(1, 16, 100, 4, 100, ctypes.byref(s), 16, 16, None) == -1


def test_sample_logits_abi_refuses_missing_outputs_and_odd_addresses(lib):
    s = sampling()
    assert lib.lce_sample_logits(1, 16, 100, 4, 100, None, 16, 16, None) == -1
    assert lib.lce_sample_logits(1, 16, 100, 4, 100, ctypes.byref(s), None, 16, None) == -1
    assert lib.lce_sample_logits(1, 16, 100, 4, 100, ctypes.byref(s), 16, None, None) == -1
    assert lib.lce_sample_logits(1, 15, 100, 4, 100, ctypes.byref(s), 16, 16, None) == -3
    assert lib.lce_sample_logits(1, 16, 100, 4, 1 << 31, ctypes.byref(s), 16, 16, None) == -8


def test_no_rows_need_no_device(lib):
    s = sampling(u=None)
    assert lib.lce_top_logits(1, None, 100, 0, 100, 8, 1.0, None, None, None, None) == 0
    assert lib.lce_sample_logits(1, None, 100, 0, 100, ctypes.byref(s), None, None, None) == 0


def test_sampling_structure_has_the_layout_of_the_header(tmp_path):
    import shutil
    import subprocess
    from pathlib import Path

    gcc = shutil.which("gcc")
    if gcc is None:
        pytest.skip("no C compiler")
    header = Path(__file__).resolve().parent.parent / "include" / "lce_b200.h"
    fields = [f[0] for f in _native.Sampling._fields_]
    lines = ['#include <stdio.h>', '#include <stddef.h>', f'#include "{header}"', "int main(void) {",
             '  printf("%zu %d %d\\n", sizeof(lce_sampling), LCE_TOP_MAX, LCE_SAMPLING_U_F64);']
    lines += [f'  printf("%zu\\n", offsetof(lce_sampling, {f}));' for f in fields] + ["  return 0;", "}"]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines))
    subprocess.run([gcc, "-std=c99", "-Wall", "-Werror", "-pedantic", "-o", str(exe), str(src)], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    assert got == ([ctypes.sizeof(_native.Sampling), _native.TOP_MAX, _native.SAMPLING_U_F64]
                   + [getattr(_native.Sampling, f).offset for f in fields])
