"""CPU check of the kernels that start while their producer still runs
(programmatic dependent launch).

A pointer declared `const T* __restrict__` lets the compiler load through the
read-only path, which is allowed only for memory that nobody writes while the
kernel lives -- and such a kernel lives while its producer writes.  So what a
producer writes must not be declared that way; what stays `__restrict__` is
named here, with the reason."""
import glob
import os
import re

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(REPO, "gpu_algos_b200", "csrc")

# inputs of the whole call, written before its first kernel (which is launched normally) starts
READ_ONLY = {
    "ortho_split_kernel": {"G"},
    "ortho_split_tall_kernel": {"G"},
    "q4_tile_kernel": {"codes", "scales"},
    "glm_finalize_kernel": {"M"},
    "glm_exchange_kernel": {"M"},
    "ortho_gemm_kernel": set(),
}


def _kernels():
    """(name, parameter list, body) of every __global__ function."""
    for path in sorted(glob.glob(os.path.join(CSRC, "*.cu")) + glob.glob(os.path.join(CSRC, "*.cuh"))):
        with open(path) as f:
            src = re.sub(r"//[^\n]*", "", f.read())
        for m in re.finditer(r"__global__\s+void\s+(?:__launch_bounds__\((?:[^()]|\([^()]*\))*\)\s*)?(\w+)\s*\(", src):
            depth, i = 1, m.end()
            while depth:
                depth += {"(": 1, ")": -1}.get(src[i], 0)
                i += 1
            params = src[m.end():i - 1]
            start = src.index("{", i)
            if ";" in src[i:start]:
                continue  # a declaration
            depth, j = 1, start + 1
            while depth:
                depth += {"{": 1, "}": -1}.get(src[j], 0)
                j += 1
            yield m.group(1), params, src[start:j]


def test_early_kernels_read_their_producers_output_with_plain_loads():
    early = {}
    for name, params, body in _kernels():
        if "pdl_wait_for_producer" in body:
            early[name] = set(re.findall(r"const\s+[^,]*?\*\s*__restrict__\s+(\w+)", params))
    assert early == READ_ONLY
