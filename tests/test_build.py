"""The native build: the same sources give the same library."""
import importlib

import pytest

build = importlib.import_module("titanic-flash-41_amd.build")

# a unit with a device variable of its own file, whose symbol carries the unit's name
SOURCE = """#include <hip/hip_runtime.h>
static __device__ int table[4];
__global__ void kernel(int* p) { p[threadIdx.x] = table[threadIdx.x & 3]; }
extern "C" int launch(int* p) { kernel<<<1, 64>>>(p); return (int)hipGetLastError(); }
"""


def test_the_library_does_not_depend_on_where_it_is_built(tmp_path):
    """Two folders of sources, two folders of objects: one library and code object, whose SHA-256 so names their sources."""
    libraries = []
    for name in ("first", "second"):
        folder = tmp_path / name
        (folder / "objects").mkdir(parents=True)
        (folder / "unit.hip").write_text(SOURCE)
        (folder / "other.hip").write_text(SOURCE.replace("launch", "launch_other").replace("kernel", "other_kernel"))
        objects = [build.compile_unit(str(folder / unit), str(folder / "objects")) for unit in ("unit.hip", "other.hip")]
        made = build.link_library(objects, str(folder / "library.so")), build.compile_code_object(str(folder / "unit.hip"), str(folder / "unit.hsaco"))
        libraries.append([open(path, "rb").read() for path in made])
    assert libraries[0] == libraries[1]


def test_units_have_names_of_their_own():
    assert len(set(build.KERNEL_UNITS)) == len(build.KERNEL_UNITS)


def test_a_broken_promise_of_the_launch_bounds_fails_the_build(tmp_path):
    """Two workgroups a CU of which one fills more than half of LDS."""
    source = """#include <hip/hip_runtime.h>
__global__ void __launch_bounds__(256, %d) kernel(int* p) {
    __shared__ int s[100 * 256];
    s[threadIdx.x * 97] = p[threadIdx.x];
    __syncthreads();
    p[threadIdx.x] = s[threadIdx.x];
}
"""
    for promised in (1, 2):
        (tmp_path / "unit.hip").write_text(source % promised)
        if promised == 1:
            build.compile_unit(str(tmp_path / "unit.hip"), str(tmp_path))
        else:
            with pytest.raises(RuntimeError, match="occupancy"):
                build.compile_unit(str(tmp_path / "unit.hip"), str(tmp_path))
