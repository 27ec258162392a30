"""What the block-scaled fp8 and expert-grouped GEMM entry points refuse, before anything reaches a GPU (no GPU needed: the
pointers are never followed)."""
import os
import re
import shutil
import struct
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
pytestmark = pytest.mark.skipif(not os.path.exists(os.path.join(ROOT, "build", "libgpumon_diag.so")), reason="needs the built diagnostics library")

P, Q, R, S = 0x10000, 0x20000, 0x30000, 0x40000  # stand-ins for device addresses


@pytest.fixture(scope="module")
def diag():
    from k8s_gpu_monitor_amd.ops import diag as d
    return d


def refused(diag, match, call, *args, **kw):
    with pytest.raises(diag.DiagError, match=match) as e:
        call(*args, **kw)
    assert e.value.code == -1


def test_quantize_refusals(diag):
    f = diag.block_quantize_launch
    refused(diag, "negative", f, P, Q, R, -1, 8)
    refused(diag, "source is", f, P, Q, R, 8, 8, dtype="fp8")
    refused(diag, "null", f, None, Q, R, 8, 8)
    refused(diag, "null", f, P, None, R, 8, 8)
    refused(diag, "null", f, P, Q, 0, 8, 8)
    refused(diag, "misaligned", f, P + 1, Q, R, 8, 8)
    refused(diag, "misaligned", f, P, Q + 8, R, 8, 8)
    refused(diag, "misaligned", f, P, Q, R + 2, 8, 8)
    refused(diag, "source row stride", f, P, Q, R, 8, 200, ld_src=199)
    refused(diag, "result row stride", f, P, Q, R, 8, 200, ld_dst=200)       # not a multiple of 16
    refused(diag, "result row stride", f, P, Q, R, 8, 200, ld_dst=192)       # shorter than 200 rounded up
    refused(diag, "result row stride", f, P, Q, R, 200, 8, transpose=True, ld_dst=192)
    refused(diag, "stride of scales", f, P, Q, R, 300, 200, ld_scales=299)
    refused(diag, "stride of scales", f, P, Q, R, 300, 200, blocks="tiles", ld_scales=1)
    refused(diag, "stride of scales", f, P, Q, R, 300, 200, blocks="tiles", transpose=True, ld_scales=2)
    refused(diag, "over 2.31", f, P, Q, R, 0x7fffffff, 8)
    refused(diag, "over 2.31", f, P, Q, R, 8, 0x7fffffff - 1022)
    refused(diag, "gmd_block_quantize_launch", f, P, Q, R, 1 << 31, 8)          # does not fit its field
    with pytest.raises(KeyError):
        f(P, Q, R, 8, 8, blocks="columns")
    f(None, None, None, 0, 128)  # a size of zero is no error
    f(None, None, None, 128, 0)


def test_gemm_block_refusals(diag):
    f = diag.gemm_block_launch
    refused(diag, "negative", f, P, R, Q, R, S, -1, 8, 16)
    refused(diag, "over 2.31", f, P, R, Q, R, S, 0x7fffffff, 8, 16)
    refused(diag, "over 2.31", f, P, R, Q, R, S, 8, 8, 0x7ffffff0)
    refused(diag, "multiples of 8", f, P, R, Q, R, S, 8, 12, 16)
    refused(diag, "multiples of 16", f, P, R, Q, R, S, 8, 8, 24)
    refused(diag, "bf16 or f32", f, P, R, Q, R, S, 8, 8, 16, out="fp8")
    for bad in ((None, R, Q, R, S), (P, R, None, R, S), (P, R, Q, R, None)):
        refused(diag, "null", f, *bad, 8, 8, 16)
    refused(diag, "scales", f, P, None, Q, R, S, 8, 8, 16)
    refused(diag, "scales", f, P, R, Q, R + 1, S, 8, 8, 16)
    refused(diag, "aligned", f, P + 8, R, Q, R, S, 8, 8, 16)
    refused(diag, "aligned", f, P, R, Q, R, S + 8, 8, 8, 16)
    refused(diag, "multiple of 16 bytes", f, P, R, Q, R, S, 8, 8, 16, lda=24)
    refused(diag, "multiple of 16 bytes", f, P, R, Q, R, S, 8, 8, 16, ldc=12)
    refused(diag, "shorter than a row", f, P, R, Q, R, S, 8, 8, 48, ldb=32)
    refused(diag, "shorter than a row", f, P, R, Q, R, S, 8, 32, 48, ldc=24)
    refused(diag, "shorter than a row", f, P, R, Q, R, S, 8, 32, 48, ldc=-32)
    refused(diag, "over 8 MiB", f, P, R, Q, R, S, 8, 8, 16, lda=(8 << 20) + 16)
    refused(diag, "over 8 MiB", f, P, R, Q, R, S, 8, 8, 16, ldc=(1 << 62) + 1024, out="f32")  # must not wrap to a small one
    refused(diag, "stride of scales", f, P, R, Q, R, S, 8, 8, 16, ld_scale_a=7)
    refused(diag, "stride of scales", f, P, R, Q, R, S, 8, 16, 16, b_blocks="rows", ld_scale_b=8)
    refused(diag, "stride of scales", f, P, R, Q, R, S, 8, 16, 400, ld_scale_b=3)
    f(None, None, None, None, None, 0, 8, 16)
    f(None, None, None, None, None, 8, 0, 16)


def test_grouped_refusals(diag):
    f = diag.grouped_gemm_launch
    size = (4, 100, 64, 64)  # groups, rows, n, k
    refused(diag, "negative", f, "forward", "bf16", P, Q, S, R, 4, -1, 64, 64)
    refused(diag, "negative", f, "forward", "bf16", P, Q, S, R, -4, 1, 64, 64)
    refused(diag, "over 2.31", f, "forward", "bf16", P, Q, S, R, 4, 0x7fffffff, 64, 64)
    refused(diag, "experts", f, "wgrad", "bf16", P, Q, S, R, (1 << 20) + 1, 8, 64, 64)
    refused(diag, "bf16 or fp8", f, "forward", "f32", P, Q, S, R, *size)
    refused(diag, "result", f, "forward", "bf16", P, Q, S, R, *size, out="mxfp8")
    refused(diag, "forward only", f, "dgrad", "fp8", P, Q, S, R, *size, scale_a=P, scale_b=P)
    refused(diag, "forward only", f, "wgrad", "fp8", P, Q, S, R, *size, scale_a=P, scale_b=P)
    refused(diag, "multiples of 8", f, "forward", "bf16", P, Q, S, R, 4, 100, 60, 64)
    refused(diag, "multiples of 8", f, "forward", "bf16", P, Q, S, R, 4, 100, 64, 60)
    refused(diag, "16 .fp8", f, "forward", "fp8", P, Q, S, R, 4, 100, 64, 72, scale_a=P, scale_b=P)
    for op in ("forward", "dgrad", "wgrad"):
        refused(diag, "offsets", f, op, "bf16", P, Q, S, None, *size)
        refused(diag, "offsets", f, op, "bf16", P, Q, S, R + 2, *size)
        refused(diag, "null", f, op, "bf16", None, Q, S, R, *size)
        refused(diag, "null", f, op, "bf16", P, None, S, R, *size)
        refused(diag, "null", f, op, "bf16", P, Q, None, R, *size)
        refused(diag, "aligned", f, op, "bf16", P, Q + 2, S, R, *size)
        refused(diag, "shorter than a row", f, op, "bf16", P, Q, S, R, *size, lda=56)
        refused(diag, "multiple of 16 bytes", f, op, "bf16", P, Q, S, R, *size, ldc=68)
        refused(diag, "expert stride", f, op, "bf16", P, Q, S, R, *size, stride_w=64 * 64 - 8)
        refused(diag, "expert stride", f, op, "bf16", P, Q, S, R, *size, stride_w=64 * 64 + 4)
    refused(diag, "scales", f, "forward", "fp8", P, Q, S, R, *size)
    refused(diag, "scales", f, "forward", "fp8", P, Q, S, R, *size, scale_a=P, scale_b=Q, ld_scale_a=99)
    refused(diag, "scales", f, "forward", "fp8", P, Q, S, R, 4, 100, 256, 256, scale_a=P, scale_b=Q, ld_scale_b=1)
    refused(diag, "scales", f, "forward", "fp8", P, Q, S, R, 4, 100, 256, 256, scale_a=P, scale_b=Q, stride_scale=3)
    refused(diag, "workgroups", f, "forward", "bf16", P, Q, S, R, 1, 1 << 30, 4 << 20, 64)
    with pytest.raises(KeyError):
        f("backward", "bf16", P, Q, S, R, *size)
    f("forward", "bf16", None, None, None, None, 4, 0, 64, 64)
    f("forward", "bf16", None, None, None, None, 0, 100, 64, 64)
    f("wgrad", "bf16", None, None, None, None, 4, 100, 0, 64)
    f("dgrad", "bf16", None, None, None, None, 4, 100, 64, 0)
    refused(diag, "null", f, "dgrad", "bf16", None, None, None, R, 4, 100, 0, 64)  # a sum over nothing is still written


def test_packed_structs_match_the_header(diag, tmp_path):
    """Sizes and the offset of every field as a C compiler lays them out."""
    if not shutil.which("g++"):
        pytest.skip("needs a C++ compiler")
    fields = {"gmd_block_quantize_t": (diag._BLOCK_QUANTIZE, "src dst scales ld_src ld_dst ld_scales rows cols src_dtype blocks transpose reserved"),
              "gmd_gemm_block_t": (diag._GEMM_BLOCK, "a b c scale_a scale_b lda ldb ldc ld_scale_a ld_scale_b m n k b_blocks out_dtype reserved"),
              "gmd_grouped_gemm_t": (diag._GROUPED_GEMM, "a b c offsets scale_a scale_b lda ldb ldc stride_w ld_scale_a ld_scale_b stride_scale op "
                                     "dtype out_dtype groups rows n k reserved")}
    src = '#include <cstdio>\n#include "gpumon_diag.h"\nint main() {\n'
    for t, (_, names) in fields.items():
        src += f'printf("%zu", sizeof({t}));\n' + "".join(f'printf(" %zu", __builtin_offsetof({t}, {n}));\n' for n in names.split()) + 'puts("");\n'
    (tmp_path / "f.cc").write_text(src + "}\n")
    subprocess.run(["g++", "-I", os.path.join(ROOT, "diag"), "-o", str(tmp_path / "f"), str(tmp_path / "f.cc")], check=True)
    lines = subprocess.run([str(tmp_path / "f")], check=True, capture_output=True, text=True).stdout.splitlines()
    import struct
    for line, (form, names) in zip(lines, fields.values()):
        size, *offsets = map(int, line.split())
        assert form.size == size
        flat = "".join(c * int(n or 1) for n, c in re.findall(r"(\d*)([Pqi])", form.format))
        assert len(flat) == len(names.split())
        at = [struct.calcsize(flat[:i]) for i in range(len(flat))]
        assert at == offsets
