"""What a call of libhipops.so launches, found without a GPU: in a process of its own the HIP runtime's launch is one that writes down the kernel's name, its
grid and its block, and nothing runs.  Pointers of such a call are numbers that nobody follows."""
import functools
import json
import os
import shutil
import subprocess
import sys
import tempfile

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

RECORDER = r"""
#include <cxxabi.h>
#include <stddef.h>
#include <stdint.h>
#include <stdio.h>
#include <stdlib.h>
#include <map>
#include <string>
struct dim3 { uint32_t x, y, z; };
struct Configuration { dim3 grid, block; size_t shared; void* stream; };
static std::map<const void*, std::string>& names() { static std::map<const void*, std::string> n; return n; }
static Configuration pushed;
static void* module[1];
extern "C" {
void** __hipRegisterFatBinary(const void*) { return module; }
void __hipUnregisterFatBinary(void**) {}
void __hipRegisterFunction(void**, const void* host, char*, const char* name, unsigned, void*, void*, dim3*, dim3*, int*) {
    char* const plain = abi::__cxa_demangle(name, nullptr, nullptr, nullptr);
    names()[host] = plain ? plain : name;
    free(plain);
}
int __hipPushCallConfiguration(dim3 grid, dim3 block, size_t shared, void* stream) { pushed = {grid, block, shared, stream}; return 0; }
int __hipPopCallConfiguration(dim3* grid, dim3* block, size_t* shared, void** stream) {
    *grid = pushed.grid, *block = pushed.block, *shared = pushed.shared, *stream = pushed.stream;
    return 0;
}
int hipLaunchKernel(const void* host, dim3 grid, dim3 block, void**, size_t, void*) {
    printf("launch %u %u %u %u %u %u %s\n", grid.x, grid.y, grid.z, block.x, block.y, block.z, names()[host].c_str());
    fflush(stdout);
    return 0;
}
int hipGetLastError() { return 0; }
}
"""

CALLER = r"""
import ctypes, json, sys
recorder = ctypes.CDLL(sys.argv[1], ctypes.RTLD_GLOBAL)  # (first in line: the library's own references go to it)
from openvino_contrib_amd import ops_capi
L = ops_capi.lib()
for name, kind, fields, args in json.load(sys.stdin):
    got = getattr(L, name)(ctypes.byref(getattr(ops_capi, kind)(**fields)), *args)
    print("status", got, L.hipops_last_error_string().decode() if got else "", flush=True)
"""


@functools.lru_cache
def _recorder():
    folder = tempfile.mkdtemp(prefix="launches-")
    source, library = os.path.join(folder, "recorder.cpp"), os.path.join(folder, "recorder.so")
    with open(source, "w") as f:
        f.write(RECORDER)
    subprocess.run([shutil.which("g++") or "g++", "-O1", "-shared", "-fPIC", source, "-o", library], check=True)
    return library


class Launch:
    def __init__(self, line):
        parts = line.split(" ", 6)
        self.grid, self.block, self.kernel = tuple(map(int, parts[:3])), tuple(map(int, parts[3:6])), parts[6].replace("(anonymous namespace)::", "")
        self.threads = 1
        for n in self.grid + self.block:
            self.threads *= n

    def __repr__(self):
        return "%s %s %s" % (self.kernel.split("(")[0], self.grid, self.block)


def launches(*calls):
    """calls: (entry point, descriptor class of ops_capi, its fields, the other arguments as numbers or None).  For each: (status, error, [Launch])."""
    env = dict(os.environ, PYTHONPATH=ROOT)
    r = subprocess.run([sys.executable, "-c", CALLER, _recorder()], input=json.dumps(calls), capture_output=True, text=True, env=env, timeout=100)
    assert r.returncode == 0, r.stderr
    found, here = [], []
    for line in r.stdout.splitlines():
        if line.startswith("launch "):
            here.append(Launch(line[7:]))
        elif line.startswith("status "):
            status, _, error = line[7:].partition(" ")
            found.append((int(status), error, here))
            here = []
    assert len(found) == len(calls)
    return found
