"""top_logits, sample_logits and linear_distillation without a GPU: what the Python layer and the C ABI refuse, before any device is touched."""
import ctypes

import pytest
import torch

from linear_cross_entropy_loss_b200 import (LinearDistillationLoss, _native, linear_distillation, linear_logits,
                                            linear_sample, linear_top_logits, sample_logits, top_logits)


@pytest.fixture(scope="module")
def lib():
    return _native.load()


@pytest.mark.parametrize("kw", [dict(k=0), dict(k=-1), dict(k=9), dict(k=3, temperature=0.0), dict(k=3, temperature=-1.0),
                                dict(k=3, temperature=float("nan")), dict(k=3, temperature=float("inf")), dict(k=3, temperature=1e-39)])
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
    (dict(vocab=0), -1), (dict(k=0), -1), (dict(t=0.0), -1), (dict(t=float("nan")), -1), (dict(values=None), -1), (dict(t=float("inf")), -1), (dict(t=1e-40), -1),
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


def check_layout(tmp_path, name, mirror, constants):
    import shutil
    import subprocess
    from pathlib import Path

    gcc = shutil.which("gcc")
    if gcc is None:
        pytest.skip("no C compiler")
    header = Path(__file__).resolve().parent.parent / "include" / "lce_b200.h"
    fields = [f[0] for f in mirror._fields_]
    lines = ['#include <stdio.h>', '#include <stddef.h>', f'#include "{header}"', "int main(void) {",
             f'  printf("%zu\\n", sizeof({name}));']
    lines += [f'  printf("%d\\n", (int){c});' for c, _ in constants]
    lines += [f'  printf("%zu\\n", offsetof({name}, {f}));' for f in fields] + ["  return 0;", "}"]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines))
    subprocess.run([gcc, "-std=c99", "-Wall", "-Werror", "-pedantic", "-o", str(exe), str(src)], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    assert got == [ctypes.sizeof(mirror)] + [v for _, v in constants] + [getattr(mirror, f).offset for f in fields]


def test_sampling_structure_has_the_layout_of_the_header(tmp_path):
    check_layout(tmp_path, "lce_sampling", _native.Sampling,
                 [("LCE_TOP_MAX", _native.TOP_MAX), ("LCE_SAMPLING_U_F64", _native.SAMPLING_U_F64)])


# ---------------------------------------------------------------------------------------------------- distillation
def distill_args(N=4, H=16, V=32, K=3):
    return dict(x=torch.zeros(N, H), teacher_logits=torch.zeros(N, K), teacher_indices=torch.zeros(N, K, dtype=torch.int64),
                At=torch.zeros(H, V))


@pytest.mark.parametrize("change", [
    dict(At=torch.zeros(15, 32)), dict(At=torch.zeros(16)), dict(At=torch.zeros(16, 0)), dict(x=torch.zeros(0, 16), teacher_logits=torch.zeros(0, 3), teacher_indices=torch.zeros(0, 3, dtype=torch.int64)),
    dict(teacher_logits=torch.zeros(5, 3)), dict(teacher_indices=torch.zeros(4, 2, dtype=torch.int64)),
    dict(teacher_indices=torch.zeros(4, 3)), dict(teacher_indices=torch.zeros(4, 3, dtype=torch.int16)),
    dict(teacher_logits=torch.zeros(4, 3, dtype=torch.float64)), dict(teacher_logits=torch.zeros(4, 0), teacher_indices=torch.zeros(4, 0, dtype=torch.int64)),
    dict(teacher_logits=torch.zeros(4, 1025), teacher_indices=torch.zeros(4, 1025, dtype=torch.int64)),
    dict(temperature=0.0), dict(temperature=-1.0), dict(temperature=float("nan")), dict(temperature=float("inf")),
    dict(logit_scale=0.0), dict(N_chunk_size=0), dict(teacher_lse=torch.zeros(3)), dict(teacher_lse=torch.zeros(4, dtype=torch.int64)),
    dict(At=torch.zeros(16, 32, dtype=torch.bfloat16)), dict(x=torch.zeros(4, 16, dtype=torch.float64), At=torch.zeros(16, 32, dtype=torch.float64)),
    dict(teacher_indices=torch.zeros(4, 3, dtype=torch.int64, device="meta")),
])
def test_linear_distillation_refuses(change):
    a = distill_args()
    a.update(change)
    with pytest.raises(AssertionError):
        linear_distillation(**a)


def test_linear_distillation_has_no_cpu_fallback():
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        linear_distillation(**distill_args())


def test_distillation_module_is_a_head():
    head = LinearDistillationLoss(16, 32, temperature=2.0, logit_scale=0.5)
    assert head.weight.shape == (16, 32) and list(head.state_dict()) == ["weight"]
    with pytest.raises(AssertionError):
        LinearDistillationLoss(16, 32, temperature=0.0)


def teacher(**kw):
    base = dict(logits=16, indices=16, lse=None, logits_ld=8, indices_ld=8, k=8, logits_dtype=_native.DTYPE_BF16,
                indices_bits=64, temperature=1.0)
    base.update(kw)
    return _native.Teacher(**base)


def distill_problem(**kw):
    base = dict(n_rows_total=1024, chunk_rows=256, hidden=256, vocab_local=4096, vocab_offset=0, ignore_index=-100,
                world=1, dtype=_native.DTYPE_BF16, monitoring=0, want_grad=1, logit_scale=1.0, z_regularization=0.0)
    base.update(kw)
    return _native.Problem(**base)


def call_distill(lib, p, t, **kw):
    a = dict(x=16, w=16, ws=16, dx=16, dw=16, res=16, loss=16)
    a.update(kw)
    return lib.lce_distill_pass(ctypes.byref(p), None if t is None else ctypes.byref(t), a["x"], 256, a["w"], 4096, a["ws"],
                                a["dx"], 256, a["dw"], 4096, a["res"], 4096, a["loss"], None)


@pytest.mark.parametrize("p_kw,t_kw,code", [
    (dict(world=2), {}, -1), (dict(vocab_offset=5), {}, -1), (dict(chunk_buffers=2), {}, -1), (dict(monitoring=1), {}, -1),
    (dict(z_regularization=0.1), {}, -1), (dict(hidden=100), {}, -2), (dict(dtype=9), {}, -1), (dict(logit_scale=0.0), {}, -1),
    ({}, dict(k=0), -1), ({}, dict(k=1025), -8), ({}, dict(temperature=0.0), -1), ({}, dict(temperature=float("nan")), -1),
    ({}, dict(temperature=float("inf")), -1), ({}, dict(logits_dtype=3), -1), ({}, dict(indices_bits=16), -1), ({}, dict(logits=None), -1),
    ({}, dict(indices=None), -1), ({}, dict(logits_ld=-1), -1), ({}, dict(indices_ld=-8), -1),
])
def test_distill_abi_refuses(lib, p_kw, t_kw, code):
    assert call_distill(lib, distill_problem(**p_kw), teacher(**t_kw)) == code


def test_distill_abi_refuses_missing_pointers(lib):
    p = distill_problem()
    assert call_distill(lib, p, None) == -1
    for name in ("x", "w", "ws", "loss"):
        assert call_distill(lib, p, teacher(), **{name: None}) == -1
    assert call_distill(lib, p, teacher(), dx=None, dw=None) == -1
    assert call_distill(lib, distill_problem(want_grad=0), teacher()) == -1


def test_distill_workspace(lib):
    out = ctypes.c_size_t(0)
    plain = ctypes.c_size_t(0)
    p = distill_problem()
    assert lib.lce_workspace_bytes(ctypes.byref(p), ctypes.byref(plain)) == 0
    sizes = []
    for k in (1, 64, 1024):
        assert lib.lce_distill_workspace_bytes(ctypes.byref(p), k, ctypes.byref(out)) == 0
        sizes.append(out.value - plain.value)
        assert out.value >= plain.value + 1024 * 16 + 256 * k * 12 + 17 * 256 * 2
    assert sizes[2] - sizes[1] == 256 * 960 * 12
    assert lib.lce_distill_workspace_bytes(ctypes.byref(p), 8, None) == -1
    assert lib.lce_distill_workspace_bytes(ctypes.byref(p), 0, ctypes.byref(out)) == -1


def test_teacher_structure_has_the_layout_of_the_header(tmp_path):
    check_layout(tmp_path, "lce_teacher", _native.Teacher, [("LCE_TEACHER_MAX", _native.TEACHER_MAX)])


@pytest.mark.parametrize("kw,code", [(dict(src=None), -1), (dict(dst=None), -1), (dict(rows=0), -1), (dict(cols=0), -1),
                                     (dict(src_ld=-1), -1), (dict(dst_ld=96), -1), (dict(dtype=5), -1), (dict(src=17), -3),
                                     (dict(dst=24), -3), (dict(dst_ld=108), -3)])
def test_align_rows_abi_refuses(lib, kw, code):
    a = dict(src=18, src_ld=101, dst=32, dst_ld=104, dtype=1, rows=4, cols=101)
    a.update(kw)
    assert lib.lce_align_rows(a["src"], a["src_ld"], a["dst"], a["dst_ld"], a["dtype"], a["rows"], a["cols"], None) == code


@pytest.mark.parametrize("kw,code", [(dict(a=None), -1), (dict(b=None), -1), (dict(f=None), -1), (dict(rows=0), -1),
                                     (dict(cols=12), -2), (dict(ld=8), -1), (dict(dtype=4), -1), (dict(a=24), -3), (dict(ld=20), -3)])
def test_grad_scale_pair_abi_refuses(lib, kw, code):
    a = dict(a=32, b=64, f=16, rows=4, cols=16, ld=16, dtype=1)
    a.update(kw)
    assert lib.lce_grad_scale_pair(a["a"], a["ld"], a["rows"], a["cols"], a["b"], 16, 4, 16, a["dtype"], a["f"], None) == code


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=7), -1), (dict(x=None), -1), (dict(w=None), -1), (dict(out=None), -1), (dict(status=None), -1), (dict(rows=0), -1),
    (dict(hidden=0), -1), (dict(vocab=0), -1), (dict(x_ld=56), -1), (dict(w_ld=96), -1), (dict(out_ld=96), -1), (dict(scale=0.0), -1),
    (dict(hidden=60, x_ld=64), -2), (dict(vocab=1 << 31, w_ld=1 << 31, out_ld=1 << 31), -8), (dict(x=24), -3), (dict(out=24), -3), (dict(w_ld=101), -3), (dict(out_ld=101), -3),
])
def test_linear_logits_abi_refuses(lib, kw, code):
    a = dict(dtype=1, x=16, x_ld=64, w=16, w_ld=104, rows=4, hidden=64, vocab=100, scale=1.0, out=16, out_ld=100, status=16)
    a.update(kw)
    assert lib.lce_linear_logits(a["dtype"], a["x"], a["x_ld"], a["w"], a["w_ld"], a["rows"], a["hidden"], a["vocab"], a["scale"],
                                 a["out"], a["out_ld"], a["status"], None) == code


def test_head_operators_refuse():
    x, At = torch.zeros(4, 16), torch.zeros(16, 32)
    for call in (lambda: linear_logits(x, torch.zeros(15, 32)), lambda: linear_logits(x, At, 0.0), lambda: linear_logits(x, At.half()),
                 lambda: linear_top_logits(x, At, 3, N_chunk_size=0), lambda: linear_logits(x.double(), At.double())):
        with pytest.raises(AssertionError):
            call()
    for call in (lambda: linear_logits(x, At), lambda: linear_top_logits(x, At, 3), lambda: linear_sample(x, At, torch.zeros(4))):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()


@pytest.mark.parametrize("t", [4.2e-39, 3.2e-39, 2.0 ** -128])
def test_top_logits_abi_refuses_temperatures_whose_scale_is_not_a_float(lib, t):
    """1 / t is one down to just above 2^-128, log2(e) / t, which the exponentials use, is not."""
    assert lib.lce_top_logits(1, 16, 100, 4, 100, 8, t, 16, 16, 16, None) == -1



@pytest.mark.parametrize("scale,t", [(1e20, 1e-30), (1e-30, 1e20), (1e25, 1e20)])
def test_a_scale_that_the_temperature_takes_out_of_range_is_refused(lib, scale, t):
    """The logits are scaled by scale / t, the gradients by scale * t: both have to be floats above zero."""
    assert call_distill(lib, distill_problem(logit_scale=scale), teacher(temperature=t)) == -1
    a = distill_args()
    with pytest.raises(AssertionError):
        linear_distillation(**a, temperature=t, logit_scale=scale)
