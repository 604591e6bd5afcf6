"""The launches of the operators over large item vocabularies, without a GPU: a small library that stands in front of HIP's launch
functions prints each launch (kernel, grid, threads) instead of making it, and the calls below go through the real C entries with
addresses that nothing reads."""
import ctypes
import json
import os
import subprocess
import sys

import pytest

RECORDER = r"""
#define _GNU_SOURCE
#include <dlfcn.h>
#include <stdio.h>
typedef struct { unsigned x, y, z; } dim3;
static dim3 grid, block;
static size_t shared;
static void *stream;
int __hipPushCallConfiguration(dim3 g, dim3 b, size_t s, void *t) { grid = g; block = b; shared = s; stream = t; return 0; }
int __hipPopCallConfiguration(dim3 *g, dim3 *b, size_t *s, void **t) { *g = grid; *b = block; *s = shared; *t = stream; return 0; }
int hipGetLastError(void) { return 0; }
int hipLaunchKernel(const void *f, dim3 g, dim3 b, void **args, size_t s, void *t) {
    Dl_info info;
    printf("%s %u %u %u %u\n", dladdr(f, &info) && info.dli_sname ? info.dli_sname : "?", g.x, g.y, g.z, b.x);
    fflush(stdout);
    return 0;
}
"""

# argv: recorder, library, [(workspace query, its sizes, entry, its arguments)] as JSON; prints each call's launches, then its status and workspace's bytes
CALLER = """
import ctypes, json, sys
recorder, path, calls = sys.argv[1:4]
ctypes.CDLL(recorder, mode=ctypes.RTLD_GLOBAL)
lib = ctypes.CDLL(path)
for query, sizes, entry, args in json.loads(calls):
    nbytes = ctypes.c_int64()
    assert getattr(lib, query)(*[ctypes.c_int64(s) for s in sizes], ctypes.byref(nbytes)) == 0
    work = 1 << 60 if nbytes.value else None
    fn = getattr(lib, entry)
    args = [work if a == "workspace" else a for a in args]
    rc = fn(*[ctypes.c_float(a) if isinstance(a, float) else ctypes.c_int64(a) if isinstance(a, int) else None for a in args])
    print("call", rc, nbytes.value, flush=True)
"""


@pytest.fixture(scope="module")
def launches(rbg, tmp_path_factory):
    """[(workspace query, its sizes, entry, its arguments)] -> per call (workspace bytes, [(kernel, x, y, z, threads)])."""
    d = tmp_path_factory.mktemp("launches")
    (d / "recorder.c").write_text(RECORDER)
    so = str(d / "recorder.so")
    subprocess.run(["gcc", "-shared", "-fPIC", "-O1", str(d / "recorder.c"), "-o", so, "-ldl"], check=True)

    def run(calls):
        got = subprocess.run([sys.executable, "-c", CALLER, so, os.path.abspath(rbg.LIB_PATH), json.dumps(calls)], capture_output=True, text=True, timeout=120)
        assert got.returncode == 0, got.stderr
        out, at = [], []
        for line in got.stdout.splitlines():
            name, *numbers = line.split()
            if name == "call":
                assert numbers[0] == "0", line
                out.append((int(numbers[1]), at))
                at = []
            else:
                at.append((name, *map(int, numbers)))
        assert len(out) == len(calls)
        return out

    return run


Z, A, B, C, D, G = (k << 56 for k in range(1, 7))  # far apart: no range of any call below reaches the next

ROWS = [1, 3, 100, 511, 512, (1 << 21) - 1, 1 << 21] + [(k << 21) + r for k in (1, 3) for r in (1, 3, 100, 511, 512)]
WIDTHS = [8191, 8192, 40982, 262144]


def forms(n, v, dtype):
    distill = [Z, v, dtype, n, v, A, B, 7, 2.0, None, C, D, None, v, "workspace", None]
    distill_grad = [Z, v, dtype, n, v, A, B, 7, 2.0, None, C, None, G, v, "workspace", None]
    logp = [Z, v, dtype, n, v, A, B, C, "workspace", None]
    preference = [Z, v, dtype, n, v, A, B, 5, C, 0.1, 0.0, None, D, D, G, v, "workspace", None]
    return [["rbg_distill_topk_workspace", [n, v], "rbg_distill_topk", distill], ["rbg_distill_topk_workspace", [n, v], "rbg_distill_topk", distill_grad],
            ["rbg_token_logp_workspace", [n, v], "rbg_token_logp", logp], ["rbg_preference_grad_workspace", [n, v], "rbg_preference_grad", preference]]


@pytest.mark.parametrize("dtype", [0, 1])
def test_no_launch_splits_rows_further_than_its_workspace(launches, dtype):
    """A call's rows go in slices of 2^21; whether workgroups share a row, each leaving 8 bytes in the workspace, is the call's decision and not
    that of its last slice, which may have few rows."""
    calls = [c for n in ROWS for v in WIDTHS for c in forms(n, v, dtype)]
    for (query, (n, v), entry, _), (nbytes, made) in zip(calls, launches(calls)):
        own = 20 * n if entry == "rbg_preference_grad" else 0  # (what that call keeps per row in front of the parts)
        rows = 0
        for name, x, y, z, threads in made:
            if "distill_part_kernel" in name or "logp_kernel" in name and "ELb1E" in name:  # x workgroups for each of y rows
                assert 8 * x * y + own <= nbytes, (entry, n, v, made)
                rows += y
            elif any(one in name for one in ("distill_eval_kernel", "distill_row_kernel", "distill_long_kernel", "logp_kernel")):
                assert x <= 1 << 21 and y == 1
                rows += x
        assert rows == n or "pair_small_kernel" in made[0][0], (entry, n, v, made)  # (that one takes every row)
