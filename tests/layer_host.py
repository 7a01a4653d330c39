"""Runs libace_layer.so's host part without a GPU: a stand-in for the HIP calls that it makes, which notes what is asked of it.  For the tests only."""
import json
import os
import shutil
import subprocess
import sys

import pytest

from superscaler_amd import layer

SHIM = r"""
#include <stddef.h>
typedef struct { unsigned x, y, z; } dim3_t;
int shim_device, shim_fail, shim_launches, shim_unprepared;
static struct { const void *kernel; int device; } set[4096];
static int sets;
int hipGetDevice(int *d) { *d = shim_device; return 0; }
int hipGetLastError(void) { return 0; }
const char *hipGetErrorString(int e) { return e ? "failed" : "ok"; }
static struct { dim3_t grid, block; size_t lds; void *stream; } next;
int __hipPushCallConfiguration(dim3_t grid, dim3_t block, size_t lds, void *stream) {
    next.grid = grid, next.block = block, next.lds = lds, next.stream = stream;
    return 0;
}
int __hipPopCallConfiguration(dim3_t *grid, dim3_t *block, size_t *lds, void **stream) {
    *grid = next.grid, *block = next.block, *lds = next.lds, *stream = next.stream;
    return 0;
}
int hipFuncSetAttribute(const void *kernel, int what, int value) {
    if (shim_fail) return 1;
    set[sets].kernel = kernel, set[sets++].device = shim_device;
    return 0;
}
/* unprepared: more LDS than a launch has by itself, and not asked for on this device */
int hipLaunchKernel(const void *kernel, dim3_t grid, dim3_t block, void **args, size_t lds, void *stream) {
    int ready = 0;
    for (int i = 0; i < sets; ++i) ready |= set[i].kernel == kernel && set[i].device == shim_device;
    shim_launches++, shim_unprepared += lds > 65536 && !ready;
    return grid.x == 0 || grid.y == 0 || grid.z == 0 || grid.y > 65535 || grid.z > 65535 || (unsigned long long)grid.x * block.x >> 32;
}
"""

CHILD = r"""
import ctypes, json, sys
shim = ctypes.CDLL(sys.argv[1], ctypes.RTLD_GLOBAL)
lib = ctypes.CDLL(sys.argv[2])
for name in ("ace_block_norm_workspace_bytes", "ace_attend_workspace_bytes", "ace_attend_backward_workspace_bytes"):
    getattr(lib, name).restype = ctypes.c_size_t
at = lambda name: ctypes.c_int.in_dll(shim, name)
out = []
for call in json.load(sys.stdin):
    at("shim_device").value, at("shim_fail").value = call["device"], call["fail"]
    at("shim_launches").value = at("shim_unprepared").value = 0
    args = []
    for a in call["args"]:
        if isinstance(a, str): args.append(bytes.fromhex(a))
        elif isinstance(a, list): args.append((ctypes.c_int64 * len(a))(*a))
        else: args.append(None if a is None else ctypes.c_void_p(a))
    rc = getattr(lib, call["name"])(*args)
    out.append({"rc": rc, "launches": at("shim_launches").value, "unprepared": at("shim_unprepared").value})
print(json.dumps(out))
"""


def call(name, *args, device=0, fail=0):
    """A call for `run`: bytes are a packed structure, lists 64-bit arrays, numbers addresses and sizes."""
    return dict(name=name, device=device, fail=fail, args=[a.hex() if isinstance(a, bytes) else a for a in args])


def run(tmp_path, calls):
    """What the calls returned and launched, one after the other in a process of their own; nothing is computed."""
    if shutil.which("gcc") is None:
        pytest.skip("no gcc")
    source, shim = tmp_path / "shim.c", tmp_path / "shim.so"
    source.write_text(SHIM)
    subprocess.run(["gcc", "-O1", "-shared", "-fPIC", str(source), "-o", str(shim)], check=True)
    done = subprocess.run([sys.executable, "-c", CHILD, str(shim), os.path.abspath(layer._LIB_PATH)], input=json.dumps(calls), capture_output=True, text=True, check=True)
    return json.loads(done.stdout)


AT = 1 << 20      # an address that nothing reads


def norm(rows=64, width=12288, per_gate=1, gate=0, dtype=1):
    """Both norms of `width`, with biases."""
    return layer._BLOCK_NORM.pack(rows, per_gate, width, dtype, 1, 1.0, 1e-5, AT, AT, gate, AT, AT, AT, AT)


def attend(batch=2, queries=512, keys=512, heads=4, kv_heads=2, dim=128, window=0, sinks=0, dtype=1):
    strides = [n * heads * dim if i == 0 else heads * dim if i == 1 else dim for n in (queries, keys, keys, queries) for i in range(3)]
    return layer._ATTEND.pack(batch, queries, keys, heads, kv_heads, dim, dtype, window, sinks, 0.125, 0, 0, *strides, *[AT] * 5)


def norm_forward(**how):
    return ("ace_block_norm_forward", norm(**how), AT, AT, AT, None)


def norm_backward(**how):
    return ("ace_block_norm_backward", norm(**how), AT, AT, AT, AT, AT, AT if how.get("gate") else None, AT, AT, AT, AT, AT, 1 << 62, None)


def attend_forward(**how):
    return ("ace_attend_forward", attend(**how), AT, 1 << 62, None)


def attend_backward(**how):
    return ("ace_attend_backward", attend(**how), AT, [1 << 20, 1024, 128], AT, AT, AT, AT, 1 << 62, None)
