"""The compiled host entries (amp_b200/_ops.so): what the file links, and that refusals reach Python."""
import subprocess
from pathlib import Path

import pytest
import torch

import amp_b200
from amp_b200 import attention, paged, rope
from amp_b200._lib import ops

SO = Path(amp_b200.__file__).parent / "_ops.so"


@pytest.fixture(scope="module")
def built(amp_lib):
    from amp_b200 import build
    build.build_host()
    return ops()


def test_one_copy_of_the_cxx_runtime(built):
    """A second libstdc++ inside the file would meet torch's in one process."""
    needed = subprocess.run(["readelf", "-d", str(SO)], capture_output=True, text=True, check=True).stdout
    assert "libstdc++.so" in needed
    out = subprocess.run(["nm", "-D", "--defined-only", str(SO)], capture_output=True, text=True, check=True).stdout
    assert [ln.split()[-1] for ln in out.splitlines() if " T " in ln] == ["PyInit__ops"]


def test_every_function_is_bound_and_declared(built):
    from amp_b200._lib import SIGNATURES
    assert set(built.names()) <= set(SIGNATURES)
    with pytest.raises(KeyError):
        built.bind({}, ValueError)
    with pytest.raises(TypeError):
        built.bind(1)
    with pytest.raises(TypeError):
        built.copy_pages(1)


X = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
I = torch.zeros(2, dtype=torch.int32)
POOL = torch.zeros(3, 2, 16, 64, dtype=torch.bfloat16)
CALLS = [lambda x: attention.flash_attn_varlen_fwd(x, X, X, I), lambda x: attention.flash_attn_varlen_bwd(x, X, X, X, X, X, I),
         lambda x: rope.rope_fwd(x, X, I, I), lambda x: rope.rope_bwd(x, X, I, I),
         lambda x: paged.rope_append(x, X, X, POOL, POOL, I, I, I, I, I), lambda x: paged.append(x, X, POOL, POOL, I, I, I),
         lambda x: paged.copy_pages(x, POOL, I, I), lambda x: paged.fork_sequences(x, POOL, I, I, I, I),
         lambda x: paged.extend_sequences(x, POOL, I, I, I), lambda x: paged.compact_pages(x, POOL, I, I),
         lambda x: paged.free_sequences(x, I, I)]


@pytest.mark.parametrize("first", [None, 3, "q", X, POOL], ids=lambda x: type(x).__name__)
@pytest.mark.parametrize("i", range(len(CALLS)))
def test_what_is_no_cuda_tensor_is_refused(i, first, built):
    for _ in range(3):
        with pytest.raises(ValueError):
            CALLS[i](first)


def test_a_flag_that_has_no_truth_value_is_an_error(built):
    with pytest.raises(ValueError):
        attention.flash_attn_varlen_fwd(X, X, X, I, scale="x")   # the tensors are looked at first


def test_a_file_for_another_torch_is_built_again(built, tmp_path, monkeypatch):
    from amp_b200 import _lib, build
    copy = tmp_path / "_ops.so"
    copy.write_bytes(SO.read_bytes())
    monkeypatch.setattr(build, "HOST_LIB", copy)
    compiled = []

    def run(cmd, **kw):
        compiled.append(cmd)
        Path(cmd[cmd.index("-o") + 1]).write_bytes(b"")
        return subprocess.CompletedProcess(cmd, 0, "", "")

    monkeypatch.setattr(build.subprocess, "run", run)
    assert build.build_host() == copy and not compiled           # this torch's, newer than its source
    monkeypatch.setattr(_lib, "host_abi", lambda: "amp_b200 host entries for another torch")
    assert build.build_host() == copy and len(compiled) == 1
    assert any("another torch" in a for a in compiled[0])


def test_a_file_for_another_torch_is_not_used(built, monkeypatch):
    from amp_b200 import _lib
    assert built.built_for() == _lib.host_abi() and torch.__version__ in built.built_for()
    monkeypatch.setattr(_lib, "_ops", None)
    monkeypatch.setattr(torch, "__version__", "0.0")
    with pytest.raises(RuntimeError, match="torch 0.0.*amp_b200.build"):
        _lib.ops()
    assert _lib._ops is None
