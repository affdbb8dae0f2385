"""CPU tests of the serving calls' boundary: struct layouts, refusals that need no device, and
a model of how attention's work is cut over workers (every tile once, no slot twice)."""
from __future__ import annotations

import ctypes as C
import os
import random
import subprocess

import pytest
import torch

from flashmlx_b200 import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def lib():
    from flashmlx_b200 import build
    build.build()
    return _lib.load()


def test_struct_layouts(tmp_path):
    prog = r"""
#include <stdio.h>
#include <stddef.h>
#include "flashmoe.h"
int main(void) {
  printf("%zu %zu %zu %zu %zu %zu %zu %zu %zu", sizeof(fm_rope_config), offsetof(fm_rope_config, theta),
         offsetof(fm_rope_config, attn_factor), sizeof(fm_cache_attn_config), offsetof(fm_cache_attn_config, q_ld),
         offsetof(fm_cache_attn_config, scale), sizeof(fm_evict_config), offsetof(fm_evict_config, budget),
         offsetof(fm_evict_config, recent));
  printf(" %d %d %d %d %d", FM_ROPE_UNSCALED, FM_ROPE_LINEAR, FM_ROPE_NTK, FM_ROPE_YARN, FM_ROPE_BANDED);
  return 0;
}
"""
    src, exe = tmp_path / "l.c", tmp_path / "l"
    src.write_text(prog)
    subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)])
    got = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True).stdout.split()]
    R, A, E = _lib.RopeConfig, _lib.CacheAttnConfig, _lib.EvictConfig
    assert got == [C.sizeof(R), R.theta.offset, R.attn_factor.offset, C.sizeof(A), A.q_ld.offset, A.scale.offset,
                   C.sizeof(E), E.budget.offset, E.recent.offset, _lib.FM_ROPE_UNSCALED, _lib.FM_ROPE_LINEAR,
                   _lib.FM_ROPE_NTK, _lib.FM_ROPE_YARN, _lib.FM_ROPE_BANDED]


def test_null_handles_are_refused(lib):
    assert lib.fm_rope(None, None, None, 0, 0, None, 0, None, 0) == _lib.FM_EINVAL
    assert lib.fm_rope_append(None, None, None, 0, 0, None, None, 0, 0, None, None, 0, 0, None, None, 0, None,
                              0) == _lib.FM_EINVAL
    assert lib.fm_attention_prefix(None, None, None, None, None, 0, None, None, None, 0, 0, None) == _lib.FM_EINVAL
    assert lib.fm_attention_scored(None, None, None, None, None, None, 0, 0, None, None) == _lib.FM_EINVAL
    assert lib.fm_cache_evict(None, None, None, None, None, None, None, 0, None, None, None, None, None) == _lib.FM_EINVAL
    assert lib.fm_serve_reserve(None, None, 0, 0) == _lib.FM_EINVAL


def test_host_tensors_are_refused(lib):
    from flashmlx_b200 import ops
    x = torch.zeros(2, 4, 64, dtype=torch.bfloat16)
    cache = torch.zeros(2, 4, 8, 64, dtype=torch.bfloat16)
    lens = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError):
        ops.rope(x, lens, 1e4)
    with pytest.raises(ValueError):
        ops.rope_append(x, x, x, lens, lens, cache, cache, 1e4)
    with pytest.raises(ValueError):
        ops.attention_prefix(x[:, None], None, None, cache, cache, lens)
    with pytest.raises(ValueError):
        ops.attention_scored(x[:, None], cache, cache, lens, torch.zeros(2, 4, 8))
    with pytest.raises(ValueError):
        ops.cache_evict(cache, cache, torch.zeros(2, 4, 8), lens, 4)


@pytest.mark.parametrize("scaling", [{"type": "dynamic", "factor": 2.0}, {"type": "linear", "factor": 2.0, "x": 1}])
def test_unknown_scalings_are_refused(scaling):
    from flashmlx_b200 import ops
    with pytest.raises(ValueError):
        ops._rope_config(64, 1e4, None, False, scaling)


def test_handles_are_bound_to_the_current_stream(monkeypatch):
    """An own handle is told a stream when it changes, a decoder's borrowed view every time (others
    bind the handle behind it)."""
    from flashmlx_b200 import ops

    class Lib:
        told = []

        def fm_set_stream(self, h, s):
            self.told.append(s)
            return _lib.FM_OK

    now = [7]
    monkeypatch.setattr(ops, "_raw_stream", lambda device: now[0])
    for borrowed, want in [(False, [7, 9]), (True, [7, 7, 9])]:
        h = ops.Handle.__new__(ops.Handle)  # as Decoder.handle() makes one
        h.lib, h.h, h.device, h._borrowed = Lib(), None, 0, borrowed
        h.lib.told = []
        now[0] = 7
        assert ops._bound(h, 0) is h and ops._bound(h, 0) is h
        now[0] = 9
        ops._bound(h, 0)
        assert h.lib.told == want
        with pytest.raises(ValueError):
            ops._bound(h, 1)
        h._borrowed, h.h = True, None  # nothing to destroy
