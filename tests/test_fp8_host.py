"""The 8-bit layers on the host: include/h3fp8.h's entry points are exported and bound,
their argument structures agree with the header, bad arguments are refused before any
device work, and the oracle's rounding is torch's own."""

from __future__ import annotations

import ctypes
import json
import re
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

from h3_flash_amd import _ext, fused_linear_fp8, quantize_fp8, quantize_fp8_weight
from h3_flash_amd.fp8 import _held_rows, _held_scales
from h3_flash_amd.fusions import fused_residual_gate_rmsnorm_modulate_fp8, fused_rmsnorm_modulate_fp8
from oracle.fp8 import dequantized, quantize_reference, scale_byte

ROOT = Path(__file__).resolve().parents[1]
HEADER = ROOT / "include" / "h3fp8.h"
STRUCTS = {
    "h3a_quantize_fp8_args": (_ext.QuantizeFp8Args, _ext.quantize_fp8),
    "h3a_rmsnorm_modulate_fp8_args": (_ext.RmsnormModulateFp8Args, _ext.rmsnorm_modulate_fp8),
    "h3a_residual_gate_rmsnorm_modulate_fp8_args": (_ext.ResidualGateRmsnormModulateFp8Args, _ext.residual_gate_rmsnorm_modulate_fp8),
    "h3a_linear_fp8_args": (_ext.LinearFp8Args, _ext.linear_fp8),
}
E4M3, E8M0, BF16 = torch.float8_e4m3fn, torch.float8_e8m0fnu, torch.bfloat16
# fake device pointers: only where a call that slipped through could not launch
host_only = pytest.mark.skipif(torch.cuda.is_available(), reason="fake device pointers: GPU-less hosts only")


@pytest.fixture(scope="module")
def lib():
    return _ext.load_library()


def test_every_declared_function_is_exported_and_bound(lib):
    names = sorted(set(re.findall(r"^H3A_API\s+\w+\s+(h3a_\w+)\s*\(", HEADER.read_text(), flags=re.M)))
    assert names == [
        "h3a_linear_fp8",
        "h3a_linear_fp8_required_workspace",
        "h3a_linear_fp8_workspace_size",
        "h3a_quantize_fp8",
        "h3a_residual_gate_rmsnorm_modulate_fp8",
        "h3a_rmsnorm_modulate_fp8",
    ]
    for name in names:
        assert hasattr(lib, name) and name in _ext.SIGNATURES, name
    text = HEADER.read_text()
    assert int(re.search(r"#define H3A_DTYPE_F8E4M3 (\d+)", text)[1]) == _ext.H3A_DTYPE_F8E4M3


@pytest.fixture(scope="module")
def c_layout(tmp_path_factory):
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    body = []
    for cname, (cls, _) in STRUCTS.items():
        fields = "".join(f'printf(", \\"{f}\\": %zu", offsetof({cname}, {f}));' for f, _ in cls._fields_)
        body.append(f'printf("\\"{cname}\\": {{\\"size\\": %zu", sizeof({cname}));{fields}printf("}}");')
    source = "#include <stddef.h>\n#include <stdio.h>\n#include \"h3fp8.h\"\nint main(void) {\nprintf(\"{\");\n"
    source += '\nprintf(",");\n'.join(body) + '\nprintf("}\\n");\nreturn 0;\n}\n'
    d = tmp_path_factory.mktemp("abi")
    (d / "layout.c").write_text(source)
    subprocess.run([cc, "-std=c11", "-Wall", "-Werror", "-I", str(ROOT / "include"), str(d / "layout.c"), "-o", str(d / "layout")], check=True)
    return json.loads(subprocess.run([str(d / "layout")], check=True, capture_output=True, text=True).stdout)


@pytest.mark.parametrize("cname", sorted(STRUCTS))
def test_structures_match_the_header(c_layout, cname):
    cls, launch = STRUCTS[cname]
    assert ctypes.sizeof(cls) == c_layout[cname]["size"]
    for field, _ in cls._fields_:
        assert getattr(cls, field).offset == c_layout[cname][field], field
    # and the packed form that a call makes: every member at its place
    packed = cls.from_buffer_copy(launch._pack(*range(1, len(cls._fields_) + 1)))
    assert [getattr(packed, f) for f, _ in cls._fields_] == list(range(1, len(cls._fields_) + 1))


P = 0x100000  # operands a MiB apart
ASK = _ext.H3A_WORKSPACE_ASK


def _quantize(**kw):
    base = dict(abi_version=_ext.ABI_VERSION, x=P, x_dtype=0, q=2 * P, scale=3 * P, rows=4, cols=64, block_rows=1, parts=1, x_stride=64,
                q_stride=64, scale_stride=16)
    return _ext.QuantizeFp8Args(**{**base, **kw})


def _norm(**kw):
    base = dict(abi_version=_ext.ABI_VERSION, x=P, q_out=2 * P, scale_out=3 * P, weight=P, w_dtype=0, scale=P, shift=P, table_dtype=0,
                scale_stride=64, shift_stride=64, table_rows=2, index=P, index_dtype=3, n_index=4, rows=4, cols=64, x_stride=64,
                q_stride=64, scale_out_stride=16, eps=1e-5)
    return _ext.RmsnormModulateFp8Args(**{**base, **kw})


def _residual(**kw):
    base = dict(abi_version=_ext.ABI_VERSION, residual=P, branch=P, hidden_out=P, q_out=2 * P, scale_out=3 * P, weight=P, w_dtype=0,
                gate=P, scale=P, shift=P, table_dtype=0, gate_stride=64, scale_stride=64, shift_stride=64, table_rows=2, index=P,
                index_dtype=3, n_index=4, rows=4, cols=64, residual_stride=64, branch_stride=64, hidden_stride=64, q_stride=64,
                scale_out_stride=16, eps=1e-5)
    return _ext.ResidualGateRmsnormModulateFp8Args(**{**base, **kw})


def _linear(**kw):
    base = dict(abi_version=_ext.ABI_VERSION, x=P, x_dtype=4, x_scale=2 * P, weight=3 * P, weight_scale=4 * P, y=5 * P, y_dtype=0, m=4,
                k=64, n=32, x_stride=64, x_scale_stride=16, weight_stride=64, weight_scale_stride=16, y_stride=32)
    return _ext.LinearFp8Args(**{**base, **kw})


def _linear8(**kw):
    return _linear(**{**dict(y_dtype=4, y_scale=6 * P, y_scale_stride=16), **kw})


INVALID, UNSUPPORTED = _ext.H3A_EINVAL, _ext.H3A_EUNSUPPORTED


@host_only
@pytest.mark.parametrize(
    "name, args, code, message",
    [
        ("h3a_quantize_fp8", _quantize(abi_version=3), INVALID, "abi_version"),
        ("h3a_quantize_fp8", _quantize(x_dtype=4), INVALID, "x dtype"),
        ("h3a_quantize_fp8", _quantize(rows=-1), INVALID, "bad extents"),
        ("h3a_quantize_fp8", _quantize(cols=0), INVALID, "bad extents"),
        ("h3a_quantize_fp8", _quantize(cols=40), UNSUPPORTED, "multiple of 16"),
        ("h3a_quantize_fp8", _quantize(block_rows=64), INVALID, "block_rows"),
        ("h3a_quantize_fp8", _quantize(parts=2), INVALID, "parts"),
        ("h3a_quantize_fp8", _quantize(block_rows=128, parts=3), INVALID, "parts"),
        ("h3a_quantize_fp8", _quantize(block_rows=128, parts=0), INVALID, "parts"),
        ("h3a_quantize_fp8", _quantize(rows=1 << 30), UNSUPPORTED, "too large"),
        ("h3a_quantize_fp8", _quantize(rows=(1 << 31) - 128, block_rows=128, cols=144, x_stride=144, q_stride=144), UNSUPPORTED, "too large"),
        ("h3a_quantize_fp8", _quantize(x=0), INVALID, "x must"),
        ("h3a_quantize_fp8", _quantize(x=P + 8), INVALID, "x must"),
        ("h3a_quantize_fp8", _quantize(x_stride=68), INVALID, "x must"),
        ("h3a_quantize_fp8", _quantize(x_stride=48), INVALID, "x must"),
        ("h3a_quantize_fp8", _quantize(q=0), INVALID, "q must"),
        ("h3a_quantize_fp8", _quantize(q_stride=72), INVALID, "q must"),
        ("h3a_quantize_fp8", _quantize(scale=3 * P + 4), INVALID, "rows of scales"),
        ("h3a_quantize_fp8", _quantize(scale_stride=8), INVALID, "rows of scales"),
        ("h3a_quantize_fp8", _quantize(cols=4096, x_stride=4096, q_stride=4096, scale_stride=16), INVALID, "rows of scales"),
        ("h3a_quantize_fp8", _quantize(q=P), INVALID, "overlap"),
        ("h3a_quantize_fp8", _quantize(scale=P + 64), INVALID, "overlap"),
        ("h3a_quantize_fp8", _quantize(scale=2 * P), INVALID, "overlap"),
        ("h3a_rmsnorm_modulate_fp8", _norm(abi_version=3), INVALID, "abi_version"),
        ("h3a_rmsnorm_modulate_fp8", _norm(cols=0), INVALID, "bad extents"),
        ("h3a_rmsnorm_modulate_fp8", _norm(cols=40), UNSUPPORTED, "multiple of 16"),
        ("h3a_rmsnorm_modulate_fp8", _norm(cols=16400, x_stride=16400, scale_stride=16400, shift_stride=16400), UNSUPPORTED, "at most 16384"),
        ("h3a_rmsnorm_modulate_fp8", _norm(rows=1 << 24), UNSUPPORTED, "too large"),
        ("h3a_rmsnorm_modulate_fp8", _norm(x=P + 2), INVALID, "aligned"),
        ("h3a_rmsnorm_modulate_fp8", _norm(weight=P + 2), INVALID, "aligned"),
        ("h3a_rmsnorm_modulate_fp8", _norm(shift_stride=66), INVALID, "aligned"),
        ("h3a_rmsnorm_modulate_fp8", _norm(x=0), INVALID, "NULL x"),
        ("h3a_rmsnorm_modulate_fp8", _norm(q_out=0), INVALID, "q_out"),
        ("h3a_rmsnorm_modulate_fp8", _norm(q_stride=40), INVALID, "q_out"),
        ("h3a_rmsnorm_modulate_fp8", _norm(scale_out=0), INVALID, "scale_out"),
        ("h3a_rmsnorm_modulate_fp8", _norm(scale_out_stride=4), INVALID, "scale_out"),
        ("h3a_rmsnorm_modulate_fp8", _norm(index_dtype=0), INVALID, "index dtype"),
        ("h3a_rmsnorm_modulate_fp8", _norm(eps=-1.0), INVALID, "eps"),
        ("h3a_residual_gate_rmsnorm_modulate_fp8", _residual(abi_version=3), INVALID, "abi_version"),
        ("h3a_residual_gate_rmsnorm_modulate_fp8", _residual(gate=0), INVALID, "table"),
        ("h3a_residual_gate_rmsnorm_modulate_fp8", _residual(branch=0), INVALID, "NULL branch"),
        ("h3a_residual_gate_rmsnorm_modulate_fp8", _residual(hidden_out=P + 2), INVALID, "aligned"),
        ("h3a_residual_gate_rmsnorm_modulate_fp8", _residual(q_out=2 * P + 8), INVALID, "q_out"),
        ("h3a_linear_fp8", _linear(abi_version=3), INVALID, "abi_version"),
        ("h3a_linear_fp8", _linear(k=0), INVALID, "bad extents"),
        ("h3a_linear_fp8", _linear(m=-1), INVALID, "bad extents"),
        ("h3a_linear_fp8", _linear(x_dtype=1), INVALID, "x dtype"),
        ("h3a_linear_fp8", _linear(y_dtype=1), INVALID, "y dtype"),
        ("h3a_linear_fp8", _linear(k=56), UNSUPPORTED, "multiple of 16"),
        ("h3a_linear_fp8", _linear(n=28), UNSUPPORTED, "of 8"),
        ("h3a_linear_fp8", _linear8(n=40, y_stride=48), UNSUPPORTED, "of 16"),
        ("h3a_linear_fp8", _linear(activation=5), INVALID, "activation"),
        ("h3a_linear_fp8", _linear(m=1 << 31), UNSUPPORTED, "too large"),
        ("h3a_linear_fp8", _linear(x=0), INVALID, "x must"),
        ("h3a_linear_fp8", _linear(x_scale=0), INVALID, "rows of scales"),
        ("h3a_linear_fp8", _linear(x_scale_stride=8), INVALID, "rows of scales"),
        ("h3a_linear_fp8", _linear(x_dtype=0, x=P + 8), INVALID, "x must"),
        ("h3a_linear_fp8", _linear(x_dtype=0, x_stride=60), INVALID, "x must"),
        ("h3a_linear_fp8", _linear(weight=3 * P + 8), INVALID, "weight must"),
        ("h3a_linear_fp8", _linear(weight_stride=72), INVALID, "weight must"),
        ("h3a_linear_fp8", _linear(weight_scale=4 * P + 8), INVALID, "rows of scales"),
        ("h3a_linear_fp8", _linear(y_stride=36), INVALID, "y must"),
        ("h3a_linear_fp8", _linear8(y_stride=40), INVALID, "y must"),
        ("h3a_linear_fp8", _linear8(y_scale=0), INVALID, "rows of scales"),
        ("h3a_linear_fp8", _linear(weight_stride=1 << 23), UNSUPPORTED, "2^31"),
        ("h3a_linear_fp8", _linear(x_dtype=0, x_stride=1 << 22), UNSUPPORTED, "2^31"),
        ("h3a_linear_fp8", _linear(x_scale_stride=1 << 23), UNSUPPORTED, "2^31"),
        ("h3a_linear_fp8", _linear(n=1 << 20, y_stride=1 << 20, weight_scale_stride=1 << 17), UNSUPPORTED, "scales of weight"),
        ("h3a_linear_fp8", _linear(y_stride=1 << 22), UNSUPPORTED, "2^31"),
        ("h3a_linear_fp8", _linear8(y_stride=1 << 23), UNSUPPORTED, "2^31"),
        ("h3a_linear_fp8", _linear8(y_scale_stride=1 << 23), UNSUPPORTED, "2^31"),
        ("h3a_linear_fp8", _linear(residual=P, residual_stride=1 << 22), UNSUPPORTED, "2^31"),
        ("h3a_linear_fp8", _linear(gate=P, gate_stride=32, table_rows=1 << 31, index=P, index_dtype=3, n_index=1), UNSUPPORTED, "2^31 rows"),
        ("h3a_linear_fp8", _linear(n=1 << 30), UNSUPPORTED, "too large"),
        ("h3a_linear_fp8", _linear(k=1 << 30), UNSUPPORTED, "too large"),
        ("h3a_linear_fp8", _linear(m=1 << 30, n=1 << 14, y_stride=1 << 14), UNSUPPORTED, "grid too large"),
        ("h3a_linear_fp8", _linear(bias=P, bias_dtype=2), INVALID, "bias dtype"),
        ("h3a_linear_fp8", _linear(bias=P + 8), INVALID, "bias"),
        ("h3a_linear_fp8", _linear(residual=P, residual_stride=24), INVALID, "residual_stride"),
        ("h3a_linear_fp8", _linear(gate=P, gate_stride=32, table_rows=1), INVALID, "index"),
        ("h3a_linear_fp8", _linear(gate=P, gate_stride=36, table_rows=1, index=P, index_dtype=3, n_index=1), INVALID, "gate rows"),
        ("h3a_linear_fp8", _linear(y=P), INVALID, "overlaps"),
        ("h3a_linear_fp8", _linear(y=3 * P + 1024), INVALID, "overlaps"),
        ("h3a_linear_fp8", _linear(y=4 * P), INVALID, "overlaps"),
        ("h3a_linear_fp8", _linear(y=2 * P + 48), INVALID, "overlaps"),
        ("h3a_linear_fp8", _linear(residual=5 * P + 16, residual_stride=32), INVALID, "overlaps"),
        ("h3a_linear_fp8", _linear8(residual=5 * P, residual_stride=32), INVALID, "overlaps"),
        ("h3a_linear_fp8", _linear8(y_scale=5 * P), INVALID, "overlaps"),
        ("h3a_linear_fp8", _linear8(y_scale=P), INVALID, "overlaps"),
        ("h3a_linear_fp8", _linear8(), INVALID, "workspace must hold"),
        ("h3a_linear_fp8", _linear8(workspace=7 * P + 128, workspace_bytes=1 << 20), INVALID, "workspace must hold"),
        ("h3a_linear_fp8", _linear8(workspace=7 * P, workspace_bytes=100), INVALID, "workspace must hold"),
    ],
)
def test_validation(lib, name, args, code, message):
    assert getattr(lib, name)(ctypes.byref(args), None) == code
    assert message in _ext.last_error(lib), _ext.last_error(lib)


@host_only
def test_null_arguments_and_empty_problems(lib):
    for name in ("h3a_quantize_fp8", "h3a_rmsnorm_modulate_fp8", "h3a_residual_gate_rmsnorm_modulate_fp8", "h3a_linear_fp8"):
        assert getattr(lib, name)(None, None) == INVALID
    assert lib.h3a_quantize_fp8(ctypes.byref(_quantize(rows=0, x=0)), None) == _ext.H3A_OK
    assert lib.h3a_rmsnorm_modulate_fp8(ctypes.byref(_norm(rows=0, x=0, q_out=0)), None) == _ext.H3A_OK
    assert lib.h3a_residual_gate_rmsnorm_modulate_fp8(ctypes.byref(_residual(rows=0, branch=0)), None) == _ext.H3A_OK
    assert lib.h3a_linear_fp8(ctypes.byref(_linear(m=0, x=0)), None) == _ext.H3A_OK


@host_only
def test_workspace_queries(lib):
    size, required = lib.h3a_linear_fp8_workspace_size, lib.h3a_linear_fp8_required_workspace
    ref = ctypes.byref
    assert size(ref(_linear())) == required(ref(_linear())) == 0
    assert required(ref(_linear8())) == size(ref(_linear8())) == 4 * 4 * 32  # the fp32 result of a few tokens
    assert lib.h3a_linear_fp8(ref(_linear8(workspace_bytes=ASK)), None) == _ext.H3A_NEED_WORKSPACE
    assert size(ref(_linear(k=40))) == UNSUPPORTED and required(None) == INVALID
    for m in (40, 300, 6240):
        bf16 = _linear(m=m, x_dtype=0, x_scale=0, k=4096, x_stride=4096, weight_stride=4096, weight_scale_stride=32, n=256, y_stride=256)
        assert size(ref(bf16)) >= required(ref(bf16)) >= 0


def test_host_tensors_never_reach_a_launch():
    x, ones = torch.zeros(4, 64, dtype=BF16), torch.ones(64, dtype=BF16)
    q, s = torch.zeros(4, 64).to(E4M3), torch.zeros(4, 1, dtype=torch.uint8).view(E8M0)
    index = torch.zeros(1, dtype=torch.int64)
    for call in (
        lambda: quantize_fp8(x),
        lambda: quantize_fp8_weight(x),
        lambda: fused_rmsnorm_modulate_fp8(x, ones, x, x, index, 1e-5),
        lambda: fused_residual_gate_rmsnorm_modulate_fp8(x, x, x, ones, x, x, index, 1e-5),
        lambda: fused_linear_fp8(x, q[:, :64].repeat(2, 1), s[:1]),
        lambda: fused_linear_fp8(q, q.repeat(2, 1), s[:1], x_scale=s),
    ):
        with pytest.raises((RuntimeError, ValueError), match="ROCm device"):
            call()


def test_refusals_of_the_wrappers():
    x, q = torch.zeros(4, 64, dtype=BF16), torch.zeros(8, 64).to(E4M3)
    s = torch.zeros(1, 1, dtype=torch.uint8).view(E8M0)
    for error, call in (
        (TypeError, lambda: quantize_fp8(x.half())),
        (TypeError, lambda: quantize_fp8_weight(q)),
        (ValueError, lambda: quantize_fp8(torch.zeros((), dtype=BF16))),
        (ValueError, lambda: quantize_fp8_weight(x[0])),
        (ValueError, lambda: quantize_fp8_weight(x[:3], gated=True)),
        (TypeError, lambda: fused_linear_fp8(x, x, s)),
        (ValueError, lambda: fused_linear_fp8(x[:, :48], q, s)),
        (ValueError, lambda: fused_linear_fp8(x, q, s, activation="tanh")),
        (ValueError, lambda: fused_linear_fp8(x, q[:7], s, gated=True)),
        (ValueError, lambda: fused_linear_fp8(x[:, :40], q[:, :40], s)),
        (ValueError, lambda: fused_linear_fp8(x, q[:4], s)),
        (ValueError, lambda: fused_linear_fp8(x, q, s, quantize=True)),  # 8 features
    ):
        with pytest.raises(error):
            call()


def test_operands_are_held_in_aligned_rows():
    buffer = torch.zeros(4096, dtype=torch.uint8)
    base = -buffer.data_ptr() % 16
    rows = buffer[base : base + 4 * 96].view(4, 96)
    held, n, stride = _held_rows(rows[:, :64], 64)
    assert (held.data_ptr(), n, stride) == (rows.data_ptr(), 4, 96)
    for moved in (rows[:, 1:65], buffer[base : base + 4 * 72].view(4, 72)[:, :64], rows.t()[:64].t()[:, ::1].t().contiguous().t()):
        held, n, stride = _held_rows(moved, moved.shape[1])
        assert held.data_ptr() % 16 == 0 and stride % 16 == 0 and held.stride(0) == stride and torch.equal(held, moved)
    scales = rows[:, :42].view(E8M0)
    held, stride = _held_scales(scales, 4, 42)
    assert (held.data_ptr(), stride) == (scales.data_ptr(), 96)
    # rows that start anywhere, and a last row whose 16 bytes the storage does not hold
    for moved in (rows[:, 1:43].view(E8M0), torch.full((4, 42), 3, dtype=torch.uint8).view(E8M0),
                  torch.zeros(48 * 3 + 42, dtype=torch.uint8).as_strided((4, 42), (48, 1)).view(E8M0)):
        held, stride = _held_scales(moved, 4, 42)
        assert stride == 48 and held.shape == (4, 48) and torch.equal(held[:, :42], moved.view(torch.uint8))


def test_the_oracle_rounds_as_torch_does():
    g = torch.Generator().manual_seed(3)
    x = torch.randn((50, 400), generator=g) * torch.exp2(torch.randint(-20, 20, (50, 1), generator=g).float())
    q, byte = quantize_reference(x)
    s = torch.exp2(byte.float() - 127).repeat_interleave(128, 1)[:, :400]
    assert torch.equal(q.float(), (x / s).to(E4M3).float())
    assert (q.abs().amax(1) > 200).all() and q.abs().max() <= 448
    assert torch.equal(scale_byte(torch.tensor([448.0, 449.0, 224.0, 0.0, 1e-45, float("inf"), 3.3e38])), torch.tensor([127, 128, 126, 1, 1, 255, 247]))
    w = x[:48].repeat(6, 1)  # 288 rows
    q, byte = quantize_reference(w, 128, 2)
    assert byte.shape == (4, 4)
    back = dequantized(q.to(E4M3), byte.to(torch.uint8).view(E8M0), 128, 2)
    assert ((back - w).abs() <= torch.maximum(2.0**-4 * w.abs().double(), 2.0**-10 * torch.exp2(byte.double() - 127).max())).all()


def test_the_tile_kernels_fit():
    """As tests/test_kernel_resources.py asks of every kernel, and one workgroup of the
    product's per CU: 160 KiB of LDS, 512 registers a lane."""

    resources = pytest.importorskip("test_kernel_resources")
    if not resources.LIB_PATH.is_file():
        pytest.skip("library not built")
    found = 0
    for co in resources.gfx950_code_objects(resources.LIB_PATH.read_bytes()):
        for k in resources.kernel_metadata(co):
            if "linear_fp8" in k[".name"] or "quantize" in k[".name"]:
                found += 1
                assert k[".private_segment_fixed_size"] == 0 and k.get(".vgpr_spill_count", 0) == 0, k[".name"]
                assert k[".group_segment_fixed_size"] <= 160 * 1024 and k[".vgpr_count"] <= 512, k[".name"]
    assert found > 10
