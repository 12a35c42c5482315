"""What the cache calls keep between calls: the status words, not the partial results."""
from __future__ import annotations

import pytest
import torch

import test_cache_api as api
from min_fa3_demo_b200 import _cabi, build, cache, min_fa3_op as op
from test_cache_api import fake  # noqa: F401  (a fixture)

BIG = 40 << 20


class Recorder:
    """Stands for the C library: says how much scratch it wants, keeps the calls."""

    def __init__(self, total, kept):
        self.total, self.kept, self.calls = total, kept, []

    def __getattr__(self, name):
        if name.endswith("_kept_workspace_bytes"):
            return lambda *sizes: self.kept
        if name.endswith("_workspace_bytes"):
            return lambda *sizes: self.total

        def call(*args):
            self.calls.append((name, args))
            return 0
        return call


@pytest.mark.parametrize("call,entry,name", [("tree", "forward_tree", "b2a_tree_fwd"), ("evict", "evict_cache", "b2a_cache_evict")])
@pytest.mark.parametrize("total", [32768, BIG])
def test_only_the_status_is_kept(fake, monkeypatch, call, entry, name, total):  # noqa: F811
    lib = Recorder(total, cache._TREE_KEPT)
    monkeypatch.setattr(_cabi, "load", lambda: lib)
    monkeypatch.setattr(op._LAST, "workspaces", {}, raising=False)
    api.FUNCTIONS[call](**api.arguments(call))
    (called, args), = lib.calls
    kept = op._LAST.workspaces[entry].untyped_storage().nbytes()
    assert kept <= op._SCRATCH_KEPT
    struct = api.Library.STRUCTS[name].from_buffer_copy(args[0])
    if total == BIG:
        assert called == name + "_with_scratch" and args[2] == total - struct.workspace_bytes and struct.workspace_bytes == kept == cache._TREE_KEPT
    else:
        assert called == name and struct.workspace_bytes == kept == total


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _cabi.load()


def test_sizes(lib):
    assert lib.b2a_tree_fwd_kept_workspace_bytes() == cache._TREE_KEPT <= op._SCRATCH_KEPT
    for batch in (1, 252, 253, 60000):
        kept = lib.b2a_cache_evict_kept_workspace_bytes(batch)
        assert 16 + 4 * batch <= kept < 16 + 4 * batch + 256
        assert lib.b2a_cache_evict_workspace_bytes(batch, 1, 4000, 9000) >= kept + batch * (4 * 4000 + 9000 // 8)
    assert lib.b2a_cache_evict_kept_workspace_bytes(0) == 0


@pytest.mark.parametrize("name", ["b2a_tree_fwd", "b2a_cache_evict"])
def test_refusals(lib, name):
    import ctypes
    struct, fields, _ = api.c_arguments(name)
    call = getattr(lib, name + "_with_scratch")

    def refused(scratch, nbytes, words, code, **change):
        args = api.filled(struct, dict(fields, **change))
        assert call(ctypes.byref(args), scratch, nbytes, None) == code and words in _cabi.last_error()
    assert call(None, 256, 1 << 30, None) == _cabi.B2A_ERR_INVALID_ARGUMENT
    refused(None, 1 << 30, "scratch must be a 16-byte aligned device pointer", _cabi.B2A_ERR_INVALID_ARGUMENT)
    refused(264, 1 << 30, "scratch must be a 16-byte aligned device pointer", _cabi.B2A_ERR_INVALID_ARGUMENT)
    if name == "b2a_cache_evict":
        refused(256, 64, "scratch has 64 bytes, need", _cabi.B2A_ERR_WORKSPACE_TOO_SMALL)
        refused(256, 1 << 30, "workspace has 8 bytes, need", _cabi.B2A_ERR_WORKSPACE_TOO_SMALL, workspace_bytes=8)

