"""CPU: operators of include/b200sp_rows.h at their borders -- what no result shows (the order of a kernel's ends, which kernel a product
goes to) and calls that have to be refused before anything is launched."""
from __future__ import annotations

import re
import types
from ctypes import c_int32
from pathlib import Path

import pytest
import torch

from test_tokens_host import _csr, _mat

SOURCES = Path(__file__).resolve().parents[1] / "ops-sparse_b200" / "csrc" / "tokens"


def _code(name):
    return re.sub(r"//[^\n]*", "", (SOURCES / name).read_text())


def _kernels(name):
    """Every kernel's body, by name."""
    code, found = _code(name), {}
    for m in re.finditer(r"__global__ void[^;{]*?\b(\w+Kernel)\(", code):
        start = code.index("{", m.end())
        found[m.group(1)] = code[start:code.index("\n}\n", start)]
    return found


@pytest.mark.parametrize("name", ["tensor.cuh", "experts_tensor.cuh", "scaled_tensor.cuh", "experts_rows.cuh"])
def test_barriers_and_loads_for_whole_warps(name):
    """Instructions that a warp's lanes have to reach together come right behind a __syncwarp()."""
    code, seen = _code(name), 0
    for m in re.finditer(r'asm volatile\(\s*"[^;]*(barrier\.cluster\.arrive|tcgen05\.ld|bar\.sync|bar\.red)', code):
        assert re.search(r"__syncwarp\(\);\s*$", code[:m.start()]), code[m.start() - 80:m.end()]
        seen += 1
    assert seen >= 1 or name == "experts_tensor.cuh"


@pytest.mark.parametrize("name,kernel", [("experts_tensor.cuh", "ExpertsTensorKernel"), ("scaled_tensor.cuh", "ScaledTensorKernel"),
                                         ("scaled_tensor.cuh", "ScaledSplitKernel")])
def test_tensor_memory_is_freed_behind_its_readers(name, kernel):
    """The last reads of tensor memory, a fence, a barrier, a fence, then it is freed."""
    body = _kernels(name)[kernel]
    end = body[body.rindex("LoadColumns32"):]
    before = re.search(r"TensorBefore\(\)|fence::before_thread_sync", end)
    assert before
    meets = re.search(r"__syncthreads\(\)|ClusterMeet\(\)|barrier\.cluster", end[before.end():])
    assert meets
    rest = end[before.end() + meets.end():]
    assert re.search(r"TensorAfter\(\)|fence::after_thread_sync", rest[:rest.index("dealloc")])


@pytest.mark.parametrize("name,kernel", [("experts_tensor.cuh", "ExpertsTensorKernel"), ("scaled_tensor.cuh", "ScaledTensorKernel")])
def test_both_ctas_of_a_pair_see_the_last_signal(name, kernel):
    """Commits of the first CTA of a pair signal barriers in both: neither ends before the last one has come in where it is."""
    body = _kernels(name)[kernel]
    end = body[body.rindex("__syncthreads()"):]
    wait = re.search(r"\n    if \(warp == 0\) [^;\n]*BarWaitWarp\(&sLast", end)  # of every CTA, outside the branches of the first
    assert wait and wait.start() < end.index("dealloc") and body.count("MmaCommit<kPair>(&sLast)") == 1


def test_the_form_of_a_product(pkg):
    """Which kernel a product goes to can be asked for, under the product's own checks."""
    f, I8, info = pkg.lib().b200spScaledMMInfo, pkg.ACL_INT8, (c_int32 * 3)()
    bad = pkg.ACL_SPARSE_STATUS_INVALID_VALUE

    def form(many, depth, channels, R=None, experts=1):
        info[:] = [-1] * 3
        assert f(R, _mat(pkg, many, depth, I8), _mat(pkg, experts * channels, depth, I8), _mat(pkg, many, channels), info) == 0
        return tuple(info)

    assert form(1, 4096, 4096) == (3, 0, 1) and form(8192, 4096, 4096)[0] == 1 and form(61, 4096, 4096)[0] == 2
    assert form(320, 512, 200)[0] == 0 and form(8192, 4096, 128)[0] != 1  # a pair has channels for both of its CTAs
    assert form(20, 64, 300, _csr(pkg, 10, 4, 20), 4) == (0, 16, 1) and form(2, 64, 300, _csr(pkg, 1, 8, 2), 8) == (3, 0, 1)
    X, W, Y = _mat(pkg, 20, 64, I8), _mat(pkg, 48, 64, I8), _mat(pkg, 20, 48)
    assert f(None, X, W, Y, None) == f(None, None, W, Y, info) == f(None, X, W, _mat(pkg, 20, 47), info) == bad
    assert f(_csr(pkg, 10, 4, 21), X, W, _mat(pkg, 20, 12), info) == bad and f(_csr(pkg, 10, 4, 20), X, W, _mat(pkg, 20, 12), info) == 0
    assert f(None, X, W, _mat(pkg, 20, 48, I8), info) == pkg.ACL_SPARSE_STATUS_NOT_SUPPORTED


def test_closed_optional_descriptors_are_refused(pkg):
    """A closed optional argument is no absent one: its NULL would say so."""
    from ops_sparse_b200 import api
    nobody = types.SimpleNamespace(_h=None, device_scalars=False)  # a call that gets as far is refused for it
    R = api.CsrMatrix(torch.zeros(3, dtype=torch.int32), torch.zeros(4, dtype=torch.int32), torch.zeros(4), 2, 4)
    X, S, Q = api.DnMat.row_major(torch.zeros(2, 8)), api.DnMat.row_major(torch.zeros(4, 8)), api.DnMat.row_major(torch.zeros(4, 8, dtype=torch.int8))
    values, starts, scales = api.DnVec(torch.zeros(4)), api.DnVec(torch.zeros(5, dtype=torch.int32)), api.DnVec(torch.zeros(4))
    gone, gone_S = api.DnVec(torch.zeros(5, dtype=torch.int32)), api.DnMat.row_major(torch.zeros(4, 8))
    gone.close()
    gone_S.close()
    calls = {  # with what is closed, and with what is not
        "offsets": [(lambda v: api.experts_dispatch(nobody, R, X, S, offsets=v), gone, starts),
                    (lambda v: api.experts_quantise(nobody, R, X, Q, scales, offsets=v), gone, starts)],
        "S": [(lambda v: api.experts_combine_grad(nobody, R, X, v, S, values), gone_S, S)],
        "d_values": [(lambda v: api.experts_combine_grad(nobody, R, X, S, S, v), gone, values)]}
    for name, some in calls.items():
        for call, closed, held in some:
            with pytest.raises(ValueError, match=f"{name} has been closed"):
                call(closed)
            for other in (held, None):
                with pytest.raises(pkg.AclSparseError, match="HANDLE_IS_NULLPTR"):
                    call(other)


@pytest.mark.parametrize("name,unit,most", [("scaled_tensor.cuh", "kTile", "kTileColsMost"), ("experts_tensor.cuh", "kMma", "kMmaColsMost")])
def test_clusters_on_tensor_memory_have_their_sms_to_themselves(name, unit, most):
    """CTAs that wait for each other must not wait for tensor memory, too: whatever the width of tiles, no other CTA with tiles in shared memory fits beside."""
    code = _code(name)
    number = lambda n: eval(re.search(rf"constexpr int {n} = ([^;]+);", code).group(1), {"kTileShared": 192 << 10, "kTileRows": 128, "kTileDepth": 128,  # noqa: E731
                                                                                       "kMmaRows": 128, "kMmaDepth": 64})
    shared, stages, first = number(f"{unit}Shared"), number(f"{unit}StagesMost"), number("kTileWBytes" if unit == "kTile" else "kMmaABytes")
    for cols in (16, 32, 64, 128, 256):
        for stage in (first + cols * 128, first + cols * 64):
            assert min(shared // stage, stages) * stage >= 160 << 10  # of 228
    if unit == "kTile":
        assert number("kSplitShared") >= 160 << 10 and "kSplitShared}" in code
