"""The block operators' C ABI on the host: the entry points that include/h3block.h
declares are exported and bound, their argument structures agree with the header,
and bad arguments are refused before any device work."""

from __future__ import annotations

import ctypes
import json
import re
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

from h3_flash_amd import _ext, fused_linear, select_key_blocks, sparse_attn_func
from h3_flash_amd.fusions import fused_rmsnorm_residual_gate_rmsnorm_modulate
from h3_flash_amd.sparse_attention import _select_workspace

ROOT = Path(__file__).resolve().parents[1]
HEADER = ROOT / "include" / "h3block.h"
STRUCTS = {
    "h3a_linear_args": (_ext.LinearArgs, _ext.linear),
    "h3a_rmsnorm_residual_gate_rmsnorm_modulate_args": (
        _ext.RmsnormResidualGateRmsnormModulateArgs,
        _ext.rmsnorm_residual_gate_rmsnorm_modulate,
    ),
    "h3a_block_select_args": (_ext.BlockSelectArgs, _ext.block_select),
    "h3a_attn_sparse_args": (_ext.AttnSparseArgs, _ext.attn_sparse),
}
# fake device pointers: only where a call that slipped through could not launch
host_only = pytest.mark.skipif(torch.cuda.is_available(), reason="fake device pointers: GPU-less hosts only")


@pytest.fixture(scope="module")
def lib():
    return _ext.load_library()


def test_every_declared_function_is_exported_and_bound(lib):
    names = sorted(set(re.findall(r"^H3A_API\s+\w+\s+(h3a_\w+)\s*\(", HEADER.read_text(), flags=re.M)))
    assert names == [
        "h3a_attn_sparse",
        "h3a_attn_sparse_workspace_size",
        "h3a_block_select",
        "h3a_block_select_workspace_size",
        "h3a_linear",
        "h3a_linear_workspace_size",
        "h3a_rmsnorm_residual_gate_rmsnorm_modulate",
    ]
    for name in names:
        assert hasattr(lib, name) and name in _ext.SIGNATURES, name


def test_constants_match_the_header():
    text = HEADER.read_text()
    value = lambda name: int(re.search(rf"#define {name} (\d+)", text)[1])  # noqa: E731
    assert value("H3A_BLOCK_Q") == _ext.H3A_BLOCK_Q and value("H3A_BLOCK_K") == _ext.H3A_BLOCK_K
    assert value("H3A_SPARSE_MAX_BLOCKS") == _ext.H3A_SPARSE_MAX_BLOCKS
    for name, code in _ext.ACTIVATIONS.items():
        assert value(f"H3A_ACT_{(name or 'none').upper()}") == code


@pytest.fixture(scope="module")
def c_layout(tmp_path_factory):
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    body = []
    for cname, (cls, _) in STRUCTS.items():
        fields = "".join(f'printf(", \\"{f}\\": %zu", offsetof({cname}, {f}));' for f, _ in cls._fields_)
        body.append(f'printf("\\"{cname}\\": {{\\"size\\": %zu", sizeof({cname}));{fields}printf("}}");')
    source = "#include <stddef.h>\n#include <stdio.h>\n#include \"h3block.h\"\nint main(void) {\nprintf(\"{\");\n"
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
    flat = sum(getattr(t, "_length_", 1) for _, t in cls._fields_)
    packed = cls.from_buffer_copy(launch._pack(*range(1, flat + 1)))
    values = [x for f, _ in cls._fields_ for x in (getattr(packed, f) if hasattr(getattr(packed, f), "_length_") else [getattr(packed, f)])]
    assert values == list(range(1, flat + 1))


P = 0x1000


def _linear(**kw):
    base = dict(abi_version=_ext.ABI_VERSION, x=P, weight=P, y=P, m=4, k=64, n=32, x_stride=64, weight_stride=64, y_stride=32)
    return _ext.LinearArgs(**{**base, **kw})


def _norm(**kw):
    base = dict(abi_version=_ext.ABI_VERSION, residual=P, branch=P, hidden_out=P, normed_out=P, branch_weight=P, weight=P,
                w_dtype=0, gate=P, scale=P, shift=P, table_dtype=0, gate_stride=64, scale_stride=64, shift_stride=64,
                table_rows=2, index=P, index_dtype=3, n_index=4, rows=4, cols=64, residual_stride=64, branch_stride=64,
                hidden_stride=64, normed_stride=64, residual_scale=1.0, eps=1e-5)
    return _ext.RmsnormResidualGateRmsnormModulateArgs(**{**base, **kw})


def _select(**kw):
    s = (300 * 256, 256, 128)
    base = dict(abi_version=_ext.ABI_VERSION, q=P, k=P, index=P, batch=1, heads=2, seqlen_q=300, seqlen_k=300, head_dim=128,
                q_stride=s, k_stride=s, topk=2, workspace=P, workspace_bytes=1 << 30)
    return _ext.BlockSelectArgs(**{**base, **kw})


def _sparse(**kw):
    s = (300 * 256, 256, 128)
    base = dict(abi_version=_ext.ABI_VERSION, q=P, k=P, v=P, o=P, lse=P, batch=1, heads=2, seqlen_q=300, seqlen_k=300,
                head_dim=128, q_stride=s, k_stride=s, v_stride=s, o_stride=s, lse_stride=(600, 300), softmax_scale=0.1,
                block_index=P, index_stride=(12, 6, 3), max_blocks=3)
    return _ext.AttnSparseArgs(**{**base, **kw})


INVALID, UNSUPPORTED = _ext.H3A_EINVAL, _ext.H3A_EUNSUPPORTED


@host_only
@pytest.mark.parametrize(
    "name, args, code, message",
    [
        ("h3a_linear", _linear(abi_version=3), INVALID, "abi_version"),
        ("h3a_linear", _linear(k=0), INVALID, "bad extents"),
        ("h3a_linear", _linear(m=-1), INVALID, "bad extents"),
        ("h3a_linear", _linear(k=60), UNSUPPORTED, "multiples of 8"),
        ("h3a_linear", _linear(n=36, y_stride=40), UNSUPPORTED, "multiples of 8"),
        ("h3a_linear", _linear(activation=5), INVALID, "activation"),
        ("h3a_linear", _linear(x=0), INVALID, "device pointers"),
        ("h3a_linear", _linear(weight=P + 8), INVALID, "device pointers"),
        ("h3a_linear", _linear(x_stride=56), INVALID, "strides"),
        ("h3a_linear", _linear(y_stride=36), INVALID, "strides"),
        ("h3a_linear", _linear(weight_stride=1 << 23), UNSUPPORTED, "2^31"),
        ("h3a_linear", _linear(m=1 << 31), UNSUPPORTED, "too large"),
        ("h3a_linear", _linear(m=1 << 30, n=1 << 14, y_stride=1 << 14), UNSUPPORTED, "grid too large"),
        ("h3a_linear", _linear(bias=P, bias_dtype=2), INVALID, "bias dtype"),
        ("h3a_linear", _linear(bias=P + 8), INVALID, "bias"),
        ("h3a_linear", _linear(residual=P, residual_stride=24), INVALID, "residual_stride"),
        ("h3a_linear", _linear(gate=P, gate_stride=32, table_rows=1), INVALID, "index"),
        ("h3a_linear", _linear(gate=P, gate_stride=32, table_rows=0, index=P, index_dtype=3, n_index=1), INVALID, "index"),
        ("h3a_linear", _linear(gate=P, gate_stride=32, table_rows=1, index=P + 4, index_dtype=3, n_index=1), INVALID, "aligned"),
        ("h3a_linear", _linear(gate=P, gate_stride=36, table_rows=1, index=P, index_dtype=3, n_index=1), INVALID, "gate rows"),
        ("h3a_rmsnorm_residual_gate_rmsnorm_modulate", _norm(abi_version=0), INVALID, "abi_version"),
        ("h3a_rmsnorm_residual_gate_rmsnorm_modulate", _norm(cols=0), INVALID, "bad extents"),
        ("h3a_rmsnorm_residual_gate_rmsnorm_modulate", _norm(rows=1 << 24), UNSUPPORTED, "too large"),
        ("h3a_rmsnorm_residual_gate_rmsnorm_modulate", _norm(eps=-1.0), INVALID, "eps"),
        ("h3a_rmsnorm_residual_gate_rmsnorm_modulate", _norm(residual_scale=float("nan")), INVALID, "residual_scale"),
        ("h3a_rmsnorm_residual_gate_rmsnorm_modulate", _norm(w_dtype=2), INVALID, "weight dtype"),
        ("h3a_rmsnorm_residual_gate_rmsnorm_modulate", _norm(table_dtype=3), INVALID, "table dtype"),
        ("h3a_rmsnorm_residual_gate_rmsnorm_modulate", _norm(hidden_out=0), INVALID, "hidden_out"),
        ("h3a_rmsnorm_residual_gate_rmsnorm_modulate", _norm(branch=P + 1), INVALID, "branch"),
        ("h3a_rmsnorm_residual_gate_rmsnorm_modulate", _norm(residual_stride=63), INVALID, "residual row stride"),
        ("h3a_rmsnorm_residual_gate_rmsnorm_modulate", _norm(weight=0), INVALID, "weights"),
        ("h3a_rmsnorm_residual_gate_rmsnorm_modulate", _norm(scale=0), INVALID, "scale"),
        ("h3a_rmsnorm_residual_gate_rmsnorm_modulate", _norm(shift_stride=8), INVALID, "shift row stride"),
        ("h3a_rmsnorm_residual_gate_rmsnorm_modulate", _norm(index=0), INVALID, "index"),
        ("h3a_rmsnorm_residual_gate_rmsnorm_modulate", _norm(index_dtype=0), INVALID, "index dtype"),
        ("h3a_block_select", _select(abi_version=1), INVALID, "abi_version"),
        ("h3a_block_select", _select(head_dim=64), UNSUPPORTED, "head_dim"),
        ("h3a_block_select", _select(heads=0), INVALID, "extent"),
        ("h3a_block_select", _select(topk=0), INVALID, "topk"),
        ("h3a_block_select", _select(topk=6), INVALID, "topk"),
        ("h3a_block_select", _select(seqlen_k=64 * 32768 + 1), UNSUPPORTED, "key blocks"),
        ("h3a_block_select", _select(batch=70000), UNSUPPORTED, "65535"),
        ("h3a_block_select", _select(seqlen_q=1 << 29, seqlen_k=64 * 32768, batch=3), UNSUPPORTED, "2^22"),
        ("h3a_block_select", _select(seqlen_q=1 << 29, seqlen_k=64 * 32768), UNSUPPORTED, "2^22"),
        ("h3a_block_select", _select(q_stride=(0, 100, 128)), INVALID, "q strides"),
        ("h3a_block_select", _select(k=P + 4), INVALID, "k must"),
        ("h3a_block_select", _select(index=0), INVALID, "index"),
        ("h3a_block_select", _select(workspace=0), INVALID, "workspace"),
        ("h3a_block_select", _select(workspace=P + 128), INVALID, "workspace"),
        ("h3a_block_select", _select(workspace_bytes=100), INVALID, "workspace"),
        ("h3a_attn_sparse", _sparse(abi_version=1), INVALID, "abi_version"),
        ("h3a_attn_sparse", _sparse(head_dim=96), UNSUPPORTED, "head_dim"),
        ("h3a_attn_sparse", _sparse(softmax_scale=0.0), INVALID, "softmax_scale"),
        ("h3a_attn_sparse", _sparse(max_blocks=-1), INVALID, "list"),
        ("h3a_attn_sparse", _sparse(max_blocks=7169), UNSUPPORTED, "list"),
        ("h3a_attn_sparse", _sparse(q=0), INVALID, "q must"),
        ("h3a_attn_sparse", _sparse(v=P + 2), INVALID, "v must"),
        ("h3a_attn_sparse", _sparse(k_stride=(0, 1864136, 128)), UNSUPPORTED, "k row stride"),
        ("h3a_attn_sparse", _sparse(o_stride=(0, 64, 128)), INVALID, "o sequence stride"),
        ("h3a_attn_sparse", _sparse(block_index=0), INVALID, "block_index"),
        ("h3a_attn_sparse", _sparse(index_stride=(1, -1, 1)), INVALID, "index strides"),
        ("h3a_attn_sparse", _sparse(block_count=P + 2), INVALID, "block_count"),
        ("h3a_attn_sparse", _sparse(lse=P + 2), INVALID, "lse"),
        ("h3a_attn_sparse", _sparse(seqlen_q=1 << 30), INVALID, "too large"),
        ("h3a_attn_sparse", _sparse(seqlen_q=1 << 28), UNSUPPORTED, "grid too large"),
    ],
)
def test_validation(lib, name, args, code, message):
    assert getattr(lib, name)(ctypes.byref(args), None) == code
    assert message in _ext.last_error(lib), _ext.last_error(lib)


@host_only
def test_null_arguments_and_empty_problems(lib):
    for name in ("h3a_linear", "h3a_rmsnorm_residual_gate_rmsnorm_modulate", "h3a_block_select", "h3a_attn_sparse"):
        assert getattr(lib, name)(None, None) == INVALID
    assert lib.h3a_linear(ctypes.byref(_linear(m=0, x=0)), None) == _ext.H3A_OK
    assert lib.h3a_rmsnorm_residual_gate_rmsnorm_modulate(ctypes.byref(_norm(rows=0, branch=0)), None) == _ext.H3A_OK
    assert lib.h3a_block_select(ctypes.byref(_select(seqlen_k=0, k=0)), None) == _ext.H3A_OK
    assert lib.h3a_attn_sparse(ctypes.byref(_sparse(seqlen_q=0, q=0)), None) == _ext.H3A_OK
    assert lib.h3a_block_select_workspace_size(ctypes.byref(_select(topk=9))) == INVALID
    # 2 heads: 2 query and 5 key blocks of 512-byte means, 2 x 5 scores, each part 256-byte aligned
    assert lib.h3a_block_select_workspace_size(ctypes.byref(_select())) == 2048 + 5120 + 256
    assert lib.h3a_attn_sparse_workspace_size(ctypes.byref(_sparse(max_blocks=8000))) == UNSUPPORTED


@host_only
@pytest.mark.parametrize("batch, heads, sq, sk", [(1, 1, 1, 1), (2, 3, 257, 65), (1, 40, 1560, 1560), (1, 5, 49920, 129024)])
def test_selection_workspace_of_the_wrapper(lib, batch, heads, sq, sk):
    args = _select(batch=batch, heads=heads, seqlen_q=sq, seqlen_k=sk, topk=1)
    want = lib.h3a_block_select_workspace_size(ctypes.byref(args))
    assert _select_workspace(batch * heads, -(-sq // 256), -(-sk // 64)) == want


def test_host_tensors_never_reach_a_launch():
    x, w = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(32, 64, dtype=torch.bfloat16)
    q, index = torch.zeros(1, 4, 1, 128, dtype=torch.bfloat16), torch.zeros(1, 1, 1, 1, dtype=torch.int32)
    for call in (
        lambda: fused_linear(x, w),
        lambda: fused_rmsnorm_residual_gate_rmsnorm_modulate(x, x, x[0], None, None, None, None, None, 1e-5),
        lambda: select_key_blocks(q, q, 1),
        lambda: sparse_attn_func(q, q, q, index),
    ):
        with pytest.raises((RuntimeError, ValueError), match="ROCm device"):
            call()


def test_sparse_kernels_fit_and_use_every_untracked_load(tmp_path):
    """The forms over lists, as tests/test_kernel_resources.py asks of the dense
    ones: a workgroup per CU, no load left in flight in registers that no path
    ahead reads."""

    resources = pytest.importorskip("test_kernel_resources")
    if not resources.LIB_PATH.is_file():
        pytest.skip("library not built")
    found = 0
    for i, co in enumerate(resources.gfx950_code_objects(resources.LIB_PATH.read_bytes())):
        path = tmp_path / f"{i}.co"
        for k in resources.kernel_metadata(co):
            name = k[".name"]
            if "attn_sparse" not in name:
                continue
            found += 1
            assert k[".vgpr_count"] + k.get(".agpr_count", 0) <= 256 and k[".max_flat_workgroup_size"] == 512, name
            assert k[".group_segment_fixed_size"] <= 160 * 1024 and k[".private_segment_fixed_size"] == 0, name
            if resources._objdump() is None:
                continue
            path.write_bytes(co)
            asm = subprocess.run([resources._objdump(), "-d", f"--disassemble-symbols={name}", str(path)], check=True,
                                 capture_output=True, text=True).stdout
            assert "buffer_load_dwordx4" in asm
            assert resources._unused_loads(asm) == [], name
    assert found == 2
