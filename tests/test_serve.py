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


# ------------------------------------------------------------------ the plan of attention over caches
@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    """The library's own planning code, built alone for the host: plan(lines) -> answers."""
    from flashmlx_b200 import build
    exe = tmp_path_factory.mktemp("plan") / "serve_plan"
    subprocess.check_call([build.nvcc(), *build.ARCH, "-std=c++17", "-I", build.INCLUDE, "-I", build.CSRC,
                           os.path.join(ROOT, "tests", "cpp", "serve_plan.cu"),
                           os.path.join(build.CSRC, "serve_plan.cu"), "-o", str(exe)])

    def ask(lines):
        r = subprocess.run([str(exe)], input="\n".join(lines) + "\n", capture_output=True, text=True, timeout=600)
        assert r.returncode == 0, r.stderr
        return r.stdout.split("\n")[:-1]

    return ask


def _weight_places(B, L, group, nkv, max_len):
    """Places of the slot weights' order (full caches, a causal prompt): every 128 keys take 2 and a
    place for each tile of 128 // group whole tokens from the first that sees them on."""
    tokens = 128 // group
    tiles = -(-L // tokens)
    n = 0
    for key0 in range(0, max_len, 128):
        n += tiles - max(key0 - (max_len - L), 0) // tokens + 2
    return n * nkv * B


@pytest.mark.parametrize("B,L,group,nkv,max_len", [
    (1, 70000, 71, 1, 2 ** 22), (1, 160000, 43, 1, 2 ** 22), (3, 100000, 65, 2, 2 ** 20), (1, 800000, 127, 1, 800000),
    (1, 70000, 100, 1, 2 ** 23)])
def test_slot_weights_beyond_their_32_bit_counts_are_refused(plan, B, L, group, nkv, max_len):
    assert _weight_places(B, L, group, nkv, max_len) >= 2 ** 31
    assert plan([f"fits {B} {L} {group * nkv} {nkv} 64 0 1 1 {max_len}"]) == ["0"]


@pytest.mark.parametrize("B,L,nh,nkv,prefix,own,scored,max_len", [
    (1, 1, 1, 1, 0, 1, 1, 1), (64, 1, 32, 4, 131072, 1, 0, 131072), (16, 1, 32, 4, 0, 1, 1, 131072),
    (1, 131072, 32, 4, 0, 1, 1, 131072), (1, 100000, 128, 1, 0, 1, 1, 100000), (4, 32768, 71, 1, 0, 1, 1, 65536),
    (65535, 1, 8, 8, 0, 1, 0, 4096), (2, 8192, 64, 8, 1048576, 1, 0, 8192), (1, 1, 16, 16, 2 ** 27, 0, 0, 0)])
def test_large_calls_are_accepted(plan, B, L, nh, nkv, prefix, own, scored, max_len):
    assert plan([f"fits {B} {L} {nh} {nkv} 128 {prefix} {own} {scored} {max_len}"]) == ["1"]


def test_counts_of_the_other_kernels_beyond_32_bits_are_refused(plan):
    full = 0x7fffff00
    lines = [f"fits 1 2000000 1 1 64 0 1 0 {2 ** 28}",      # tcgen05, own caches: 7813 items of 2^21 tiles
             f"fits 500 4000 1 1 64 {2 ** 28} 0 0 0",       # tcgen05, prefix
             f"fits 1 64 1 1 64 0 1 0 {full}",              # split: four row tiles of 2^27 tiles, accepted
             f"fits 2 32 1 1 64 {full} 1 0 {full // 2}"]    # split, both sources: 2^29 + 2^28
    assert plan(lines) == ["0", "0", "1", "1"]


@pytest.mark.parametrize("steps,waits", [
    ("c c c", "| | |"),                                       # one stream: nothing
    ("c b1 c b1 c b2 c b1 c", "| | 1<0 | | 2<1 | 1<2"),       # each change waits once
    ("b1 b2 c b1 c", "| | 1<2"),                              # a stream without calls is not waited for
    ("c b1 b2 b3 c b0 c", "| | 3<0 | 0<3"),                   # bound over, the calls stay to be waited for
    ("c b1 b0 c b1 c", "| | | 1<0"),                          # back again: its own calls
    ("c b1 +1 c c -1 c b0 c", "| | | | 1<0 | 0<1"),           # a capture waits for nothing; the first call after it does
    ("c b1 +1 c b2 c -1 b0 c", "| | | 2<0 | 0<1 0<2"),        # a stream being captured is waited for later
    ("c +0 c b1 c -0 c c", "| | | | 1<0 |"),                  # the stream of earlier calls is captured itself
    ("c b1 s b2 c", "| | 1<0 |"),                             # synchronized: nothing is in flight
    ("c b1 +0 s b2 c -0 c", "| | | | 2<0"),
    ("+1 *2 b1 c b2 c c b1 c -1 -2 b2 c", "| | 2<1 | 2<1 | 1<2 | 2<1"),  # branches of one capture
    ("c b1 +1 c b2 +2 c b1 c -1 -2 c", "| | | | | 1<0 1<2"),    # two captures at a time
    ("c b1 c b2 f2 c c b1 c c", "| | 1<0 | 2<1 | | error | 1<2"),
    ("c b1 f1 c c", "| | error | 1<0"),                       # an error leaves it to be waited for
])
def test_calls_of_a_handle_on_several_streams_wait_for_one_another(plan, steps, waits):
    n = steps.split()
    assert plan([f"order {len(n)} {steps}"])[0].split() == waits.split()


@pytest.mark.parametrize("seed", [random.Random(s).randrange(2 ** 31) for s in range(8)])
def test_attention_work_is_cut_without_gaps(plan, seed):
    """Random calls: every tile of every item belongs to one worker, every piece has a slot of its own inside the
    planned workspace, where the kernels that join an item's pieces look for it; the reservation covers
    the plan."""
    assert plan([f"cut {seed} 400"]) == ["ok"]


def test_division_by_multiplication_is_exact(plan):
    assert plan(["divide 200000"]) == ["ok"]


def test_evictions_share_a_head_among_as_many_ctas_as_run_at_a_time(plan):
    """148 SMs hold 74 clusters of two and 33 of four: the 34th head would wait for a second round."""
    lines = [f"evict {heads} {n} 74 33" for heads, n in [(1, 14335), (1, 14336), (33, 2 ** 20), (34, 18431), (34, 18432), (74, 20480), (75, 20480)]]
    assert plan(lines) == ["1", "4", "4", "1", "2", "2", "1"]
    assert plan(["evict 1 20480 0 0", "evict 5 20480 5 4"]) == ["1", "2"]
