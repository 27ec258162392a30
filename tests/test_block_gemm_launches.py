"""What the block-scaled fp8 and expert-grouped GEMM entry points launch, and on which device's memory, with a stand-in for the HIP
runtime (tests/stubs/hip_stub.cc: two devices, launches are printed and reach no GPU)."""
import json
import os
import shutil
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
pytestmark = pytest.mark.skipif(not os.path.exists(os.path.join(ROOT, "build", "libgpumon_diag.so")) or not shutil.which("g++"),
                                reason="needs the built diagnostics library and g++")

CALLS = r"""
import json, sys
from k8s_gpu_monitor_amd.ops import diag
for name, args, kw in json.loads(sys.argv[1]):
    print("call", flush=True)
    try:
        getattr(diag, name)(*args, **kw)
    except diag.DiagError as e:
        print("refused", e.code, e, flush=True)
"""


@pytest.fixture(scope="module")
def stub(tmp_path_factory):
    lib = tmp_path_factory.mktemp("hip_stub") / "libhip_stub.so"
    subprocess.run(["g++", "-shared", "-fPIC", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", os.path.join(ROOT, "tests", "stubs", "hip_stub.cc"),
                    "-o", str(lib)], check=True, timeout=120)
    return lib


def run_all(stub, calls):
    """For each (function, arguments, keywords): its launches, as (grid, block), or ["refused ..."]."""
    env = dict(os.environ, PYTHONPATH=ROOT, LD_PRELOAD=" ".join(x for x in (str(stub), os.environ.get("LD_PRELOAD", "")) if x))
    r = subprocess.run([sys.executable, "-c", CALLS, json.dumps(calls)], capture_output=True, text=True, timeout=120, env=env)
    assert r.returncode == 0, r.stderr[-800:]
    out = []
    for lines in r.stdout.split("call\n")[1:]:
        out.append([])
        for line in lines.splitlines():
            if line.startswith("launch"):
                grid, block = line[len("launch "):].split(" x ")
                line = (tuple(map(int, grid.split())), tuple(map(int, block.split())))
            out[-1].append(line)
    return out


def run(stub, calls):
    """The same where each call has one launch."""
    answers = run_all(stub, calls)
    assert all(len(a) == 1 for a in answers)
    return [a[0] for a in answers]


P, AWAY = 0x10000, 1 << 32  # memory of device 0, and what has to be added for device 1


def test_operands_scales_and_offsets_of_another_device_are_refused(stub):
    calls, names = [], []

    def each(name, pointers, args, kw=(), more=()):
        """The call as it is, and with one of its pointers on the other device."""
        for away in (None, *range(len(pointers)), *more):
            p = [P + 0x10000 * i + (AWAY if i == away else 0) for i in range(len(pointers))]
            k = dict(kw, **{x: 0x900000 + 0x10000 * i + (AWAY if x == away else 0) for i, x in enumerate(more)})
            calls.append((name, [*p, *args], k))
            names.append((name, dict(kw), away))

    for blocks, transpose in (("rows", False), ("tiles", True)):
        each("block_quantize_launch", "src dst scales".split(), (64, 64), {"blocks": blocks, "transpose": transpose})
    each("gemm_block_launch", "a sa b sb c".split(), (8, 8, 16))
    for op, dtype, more in (("forward", "bf16", ()), ("dgrad", "bf16", ()), ("wgrad", "bf16", ()), ("forward", "fp8", ("scale_a", "scale_b"))):
        first = len(calls)
        each("grouped_gemm_launch", "a b c offsets".split(), (2, 64, 64, 64), more=more)
        for c in calls[first:]:
            c[1][:0] = [op, dtype]
    for (name, kw, away), got in zip(names, run(stub, calls)):
        if away is None:
            assert isinstance(got, tuple), (name, kw, got)
        else:
            assert isinstance(got, str) and got.startswith("refused -1") and "another device" in got, (name, kw, away, got)


def threads(launch):
    (gx, gy, gz), (bx, by, bz) = launch
    assert gx * bx < 1 << 32 and gy == gz == by == bz == 1
    return gx * bx


def test_no_launch_has_four_billion_threads(stub):
    """Sizes up to 2^31 - 1024: a quantisation is split into bands, a product over the limit is refused by name, and one just under it,
    or walked by a workgroup a CU, is launched."""
    most = 0x7fffffff - 1023
    q = [("block_quantize_launch", [P, 2 * P, 3 * P, rows, cols], dict(blocks=blocks, transpose=trans, dtype=dtype))
         for blocks in ("rows", "tiles") for trans in (False, True) for dtype in ("bf16", "f32")
         for rows, cols in ((1 << 27, 64), ((1 << 27) - 8, 64), (1 << 20, 1 << 20), (128, most), (most, 128), (129, most), (most, 1))]
    for call, got in zip(q, run_all(stub, q)):
        rows, cols = call[1][3:]
        by_rows = call[2]["blocks"] == "rows" and not call[2]["transpose"]
        groups = -(-rows // 8) * -(-cols // 512) if by_rows else -(-rows // 128) * -(-cols // 128)
        assert all(isinstance(x, tuple) for x in got), (call, got)
        assert sum(threads(x) for x in got) == groups * 256, (call, got)
        assert len(got) == 1 or groups * 256 >= 1 << 32
    gemm = ("gemm_block_launch", [P, 2 * P, 3 * P, 4 * P, 5 * P])
    grouped = ("grouped_gemm_launch", [P, 2 * P, 3 * P, 4 * P])

    def product(m, n, k, **kw):
        return gemm[0], [*gemm[1], m, n, k], kw

    def experts(op, *size, **kw):
        return grouped[0], [op, kw.pop("dtype", "bf16"), *grouped[1], *size], kw

    over = [product(1 << 30, 8, 16), product(most, 64, 128, b_blocks="rows"),
            experts("wgrad", 1 << 20, 1024, 8, 8), experts("forward", 1 << 20, 1 << 20, 512, 8), experts("dgrad", 1 << 20, 1 << 20, 8, 1024),
            experts("forward", 1 << 20, 1 << 20, 512, 16, dtype="fp8", scale_a=P, scale_b=P)]
    fit = [product(1 << 30, 8, 16, out="f32"), product((1 << 29) - 128, 8, 16), product(1 << 17, 1 << 16, 4096), experts("wgrad", 1 << 19, 1024, 8, 8), experts("forward", 1 << 18, 1 << 18, 512, 8),
           experts("wgrad", 1 << 14, 1 << 24, 2048, 2048), experts("dgrad", 1 << 18, 1 << 18, 8, 512)]
    for call, got in zip(over, run(stub, over)):
        assert isinstance(got, str) and got.startswith("refused -1") and "do not fit into one launch" in got, (call, got)
    for call, got in zip(fit, run(stub, fit)):
        assert isinstance(got, tuple) and threads(got), (call, got)
