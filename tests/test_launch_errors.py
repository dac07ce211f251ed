"""Calls whose launches the runtime refuses say so.  A library of launches that fail when they are told to stands in the runtime's place, in a process of its own,
so nothing here needs or reaches a device."""
import json
import subprocess
import sys

import pytest

from sensenova_u1_amd import ops
from sensenova_u1_amd.build import LIB_PATH

E_LAUNCH = -5

RUNTIME = r"""
typedef struct { unsigned x, y, z; } dim3_t;
static int error, count, bad = -1;
void fail(int which, int pending) { bad = which, count = 0, error = pending; }
int launches(void) { return count; }
int __hipPushCallConfiguration(dim3_t grid, dim3_t block, unsigned long lds, void* stream) { return 0; }
int __hipPopCallConfiguration(dim3_t* grid, dim3_t* block, unsigned long* lds, void** stream) {
    grid->x = grid->y = grid->z = block->x = block->y = block->z = 1, *lds = 0, *stream = 0;
    return 0;
}
int hipLaunchKernel(const void* f, dim3_t grid, dim3_t block, void** args, unsigned long lds, void* stream) { return count++ == bad ? (error = 1) : 0; }
int hipGetLastError(void) { const int e = error; error = 0; return e; }
"""

PROGRAM = r"""
import ctypes, json, struct, sys
runtime = ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)
lib = ctypes.CDLL(sys.argv[2])
room = ctypes.create_string_buffer(1 << 20)
P = (ctypes.addressof(room) + 255) // 256 * 256
V, I = ctypes.c_void_p, ctypes.c_int64
tables = struct.pack("5P4q", P, P + 256, P + 512, P + 768, P + 1024, 4, 4, 8, 16)       # 4 sequences of 4 pages, a ring of 8
outputs = [V(P + 2048 + (i << 16)) for i in range(6)]                                      # ends, lens, cursor, positions, slots, missing
outputs[1:3] = [V(P + 256), V(P + 1024)]


def append(tokens):
    need = lib.sngguf_page_append_workspace_bytes(I(4), I(tokens))
    return lib.sngguf_page_append(tables, V(P + 1280), I(tokens), *outputs, V(P + (7 << 16)) if need else None, I(need), None)


calls = {"append": lambda: append(4), "append in two launches": lambda: append(5000), "append without rows": lambda: append(0),
         "release": lambda: lib.sngguf_page_release(tables, V(P + 1280), None), "fork": lambda: lib.sngguf_page_fork(tables, V(P + 1280), V(P + 1536), None)}
out = {}
for name, call in calls.items():
    out[name] = []
    for bad, pending in ((-1, 0), (0, 0), (1, 0), (-1, 1)):
        runtime.fail(bad, pending)
        out[name].append([call(), runtime.launches()])
print(json.dumps(out))
"""


@pytest.fixture(scope="module")
def results(tmp_path_factory):
    ops.load_library()
    folder = tmp_path_factory.mktemp("runtime")
    (folder / "runtime.c").write_text(RUNTIME)
    subprocess.run(["gcc", "-shared", "-fPIC", "-O1", "-o", str(folder / "runtime.so"), str(folder / "runtime.c")], check=True)
    run = subprocess.run([sys.executable, "-c", PROGRAM, str(folder / "runtime.so"), LIB_PATH], check=True, capture_output=True, text=True, timeout=100)
    return json.loads(run.stdout)


# (result, launches): nothing fails; the first launch does; the second does; an error from before the call is still there
@pytest.mark.parametrize("call,launches", [("append", 1), ("append without rows", 1), ("append in two launches", 2), ("release", 1), ("fork", 1)])
def test_page_tables(results, call, launches):
    good, first, second, before = results[call]
    assert good == [0, launches]
    assert first == [E_LAUNCH, 1]
    assert second == ([E_LAUNCH, 2] if launches == 2 else [0, 1])
    assert before == [E_LAUNCH, 1]
