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


def run(stub, calls):
    """For each (function, arguments, keywords): "refused ..." or the launch, as (grid, block)."""
    env = dict(os.environ, PYTHONPATH=ROOT, LD_PRELOAD=" ".join(x for x in (str(stub), os.environ.get("LD_PRELOAD", "")) if x))
    r = subprocess.run([sys.executable, "-c", CALLS, json.dumps(calls)], capture_output=True, text=True, timeout=120, env=env)
    assert r.returncode == 0, r.stderr[-800:]
    out = []
    for lines in r.stdout.split("call\n")[1:]:
        (line,) = lines.splitlines()  # one answer to each call
        if line.startswith("launch"):
            grid, block = line[len("launch "):].split(" x ")
            out.append((tuple(map(int, grid.split())), tuple(map(int, block.split()))))
        else:
            out.append(line)
    return out


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
