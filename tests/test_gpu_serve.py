"""The serving operators (fm_rope, fm_rope_append, fm_attention_prefix, fm_attention_scored,
fm_cache_evict) on a B200 against the plain 64-bit implementations of tests/serve_util.py,
with the tolerances derived there; moves and lengths are exact."""
from __future__ import annotations

import pytest
import torch

from tests import serve_util as R

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


@pytest.fixture(autouse=True)
def _clean_status():
    """No call leaves a device-side report unless its test expects and reads it."""
    yield
    from flashmlx_b200 import ops
    ops.synchronize()


def rnd(seed, *shape, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * std).to(BF).cuda()


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def held(got, want, tol, what=""):
    err = (got.double().cpu() - want).abs()
    assert torch.isfinite(got).all(), what
    bad = err > tol
    assert not bad.any(), f"{what}: {int(bad.sum())} outside, worst {float((err / tol.clamp_min(1e-300)).max()):.2f} times the tolerance"


# ------------------------------------------------------------------ refusals (host side, nothing launched)
def refused(call, status=None):
    from flashmlx_b200 import _lib
    with pytest.raises((ValueError, TypeError, NotImplementedError, _lib.FlashMoEError)) as e:
        call()
    if isinstance(e.value, _lib.FlashMoEError) and status is not None:
        assert e.value.status == status


def test_rope_refusals():
    from flashmlx_b200 import _lib, ops
    x, p = rnd(1, 3, 2, 64), i32([0, 1, 2])
    bad = [
        lambda: ops.rope(x.float(), p, 1e4), lambda: ops.rope(x.half(), p, 1e4), lambda: ops.rope(x, p.long(), 1e4),
        lambda: ops.rope(x, p[:2], 1e4), lambda: ops.rope(x, p, 1e4, rotary_dim=3),
        lambda: ops.rope(x, p, 1e4, rotary_dim=66), lambda: ops.rope(x, p, 0.0), lambda: ops.rope(x, p, float("nan")),
        lambda: ops.rope(x, p, 1e4, scaling={"type": "linear", "factor": 0.5}),
        lambda: ops.rope(x, p, 1e4, rotary_dim=2, scaling={"type": "ntk", "factor": 2.0}),
        lambda: ops.rope(x, p, 1e4, scaling={"type": "yarn", "factor": 2.0, "original_len": 0}),
        lambda: ops.rope(x, p, 1e4, scaling={"type": "banded", "factor": 2.0, "original_len": 64, "low_freq": 4.0,
                                             "high_freq": 4.0}),
        lambda: ops.rope(rnd(1, 3, 2, 60), p, 1e4),            # head size not a multiple of 8
        lambda: ops.rope(x.transpose(1, 2).contiguous().transpose(1, 2), p, 1e4),  # heads not side by side
        lambda: ops.rope(x, p, 1e4, out=torch.empty(3, 2, 32, dtype=BF, device="cuda")),
        lambda: ops.rope(rnd(1, 4, 2, 64)[:3], p, 1e4, out=rnd(1, 3, 2, 64).float()),
    ]
    base = rnd(2, 4, 2, 64)
    bad.append(lambda: ops.rope(base[:3], p, 1e4, out=base[1:]))  # partly overlapping
    wide = rnd(3, 3 * 140)[: 3 * 132].view(3, 132)
    bad.append(lambda: ops.rope(wide[:, :128].view(3, 2, 64), p, 1e4))  # a row stride that is no multiple of 8
    for call in bad:
        refused(call, _lib.FM_EINVAL if call is not bad[12] else _lib.FM_EUNSUPPORTED)


def test_attention_refusals():
    from flashmlx_b200 import _lib, ops
    q, ck, lens = rnd(4, 2, 1, 4, 64), rnd(5, 2, 2, 16, 64), i32([3, 4])
    pk = rnd(6, 2, 8, 64)
    acc = torch.zeros(2, 2, 16, device="cuda")
    h = ops.default_handle()
    cfg = _lib.CacheAttnConfig(4, 2, 64, 16, 8, 0, 0.0)
    for call in [
        lambda: ops.attention_prefix(q, None, None), lambda: ops.attention_prefix(q, pk, pk, ck, ck, None),
        lambda: ops.attention_prefix(q, pk, pk[:1], ck, ck, lens), lambda: ops.attention_prefix(q, pk, pk, prefix_len=9),
        lambda: ops.attention_prefix(q, pk, pk, prefix_len=-1), lambda: ops.attention_prefix(q, pk, pk, lens=lens),
        lambda: ops.attention_prefix(q[:1], pk, pk, ck, ck, lens), lambda: ops.attention_prefix(q.half(), pk, pk, ck, ck, lens),
        lambda: ops.attention_prefix(rnd(7, 2, 1, 4, 32), rnd(7, 2, 8, 32), rnd(7, 2, 8, 32)),  # head size 32
        lambda: ops.attention_prefix(rnd(7, 2, 1, 3, 64), pk, pk, ck, ck, lens),                # 3 heads over 2
        lambda: ops.attention_prefix(q, pk, pk, ck, ck, lens, scale=float("nan")),
        lambda: ops.attention_scored(q, ck, ck, lens.long(), acc), lambda: ops.attention_scored(q, ck, ck, lens, acc[:1]),
        lambda: ops.attention_scored(q, ck, ck, lens, acc.half()), lambda: ops.attention_scored(q, ck, ck[:, :1], lens, acc),
        lambda: h.check(h.lib.fm_attention_prefix(h.h, _lib.C.byref(cfg), q.data_ptr(), None, None, 4, None, None, None, 2, 1,
                                                  q.data_ptr())),
        lambda: h.check(h.lib.fm_attention_prefix(h.h, _lib.C.byref(cfg), q.data_ptr(), pk.data_ptr(), pk.data_ptr(), 4, None,
                                                  None, None, 2, 1, q.data_ptr())),  # out is q
        lambda: h.check(h.lib.fm_attention_prefix(h.h, _lib.C.byref(cfg), q.data_ptr() + 2, pk.data_ptr(), pk.data_ptr(), 4,
                                                  None, None, None, 2, 1, ck.data_ptr())),
        lambda: h.check(h.lib.fm_serve_reserve(h.h, _lib.C.byref(cfg), -1, 1)),
        lambda: ops.attention_scored(rnd(7, 1, 1, 129, 64), ck[:1, :1].contiguous(), ck[:1, :1].contiguous(), lens[:1].contiguous(),
                                     acc[:1, :1].contiguous()),
    ]:
        refused(call)


def test_evict_refusals():
    from flashmlx_b200 import ops
    ck, cv, acc, lens = rnd(8, 2, 2, 16, 64), rnd(9, 2, 2, 16, 64), torch.zeros(2, 2, 16, device="cuda"), i32([9, 16])
    pos = torch.zeros(2, 2, 16, dtype=torch.int32, device="cuda")
    small = (rnd(1, 2, 2, 3, 64), rnd(1, 2, 2, 3, 64), torch.zeros(2, 2, 3, device="cuda"), None)
    other = torch.zeros_like(acc)
    for call in [
        lambda: ops.cache_evict(ck, cv, acc, lens, 0), lambda: ops.cache_evict(ck, cv, acc, lens, 4, sinks=3, recent=2),
        lambda: ops.cache_evict(ck, cv, acc, lens, 4, sinks=-1), lambda: ops.cache_evict(ck, cv, acc, lens, 4, out=small),
        lambda: ops.cache_evict(ck, cv, acc, lens, 4, out=(ck, cv, other, None)),      # half in place
        lambda: ops.cache_evict(ck, cv, acc, lens, 4, out=(cv, ck, acc, None)),        # crosswise
        lambda: ops.cache_evict(ck, cv, acc, lens, 4, positions=pos, out=(ck, cv, acc, None)),
        lambda: ops.cache_evict(ck, cv, acc.double(), lens, 4), lambda: ops.cache_evict(ck, cv, acc, lens[:1], 4),
        lambda: ops.cache_evict(ck, cv[:1], acc, lens, 4),
        lambda: ops.cache_evict(ck[:, :, ::2], cv[:, :, ::2], acc[:, :, :8].contiguous(), lens, 4),
    ]:
        refused(call)


def test_tokens_that_share_memory_are_refused():
    """A token's rows expanded over the batch have a stride of zero, which is no packed row."""
    from flashmlx_b200 import ops
    one, ck, cv, lens = rnd(10, 1, 1, 4, 64), rnd(11, 3, 2, 16, 64), rnd(12, 3, 2, 16, 64), i32([3, 4, 5])
    acc = torch.zeros(3, 2, 16, device="cuda")
    q = one.expand(3, 1, 4, 64)
    for call in [
        lambda: ops.attention_prefix(q, None, None, ck, cv, lens), lambda: ops.attention_scored(q, ck, cv, lens, acc),
        lambda: ops.attention_prefix(one.expand(3, 2, 4, 64), None, None, ck, cv, lens),
        lambda: ops.attention_prefix(q, ck[0], cv[0]), lambda: ops.rope(one[0].expand(3, 4, 64), lens, 1e4),
        lambda: ops.rope(rnd(13, 3, 4, 64), lens, 1e4, out=one[0].expand(3, 4, 64)),
        lambda: ops.attention_prefix(rnd(14, 1000).as_strided((3, 1, 4, 64), (128, 128, 64, 1)), None, None, ck, cv, lens),
    ]:
        refused(call)


def test_overlapping_memory_is_refused():
    from flashmlx_b200 import _lib, ops
    qkv, ck, cv, at = rnd(15, 2, 8, 64), rnd(16, 2, 2, 16, 64), rnd(17, 2, 2, 16, 64), i32([0, 1])
    q, k, v = qkv[:, :4], qkv[:, 4:6], qkv[:, 6:]
    rows = ck.view(2, 32, 64)
    for call in [
        lambda: ops.rope_append(q, k, v, at, at, ck, ck, 1e4), lambda: ops.rope_append(q, k, v, at, at, ck, cv, 1e4, out=qkv[:, 1:5]),
        lambda: ops.rope_append(k, k, v, at, at, ck, cv, 1e4, out=k), lambda: ops.rope_append(q, k, v, at, at, ck, cv, 1e4, out=qkv[:, 4:]),
        lambda: ops.rope_append(q, rows[:, :2], rows[:, 2:4], at, at, ck, cv, 1e4),
        lambda: ops.rope_append(q, k, v, at, at, ck, cv, 1e4, out=rows[:, :4]),
        lambda: ops.rope(qkv[:, :4], at, 1e4, out=qkv[:, 2:6]),
    ]:
        refused(call, _lib.FM_EINVAL)
    want = ops.rope(q, at, 1e4)
    assert torch.equal(ops.rope(q, at, 1e4, out=qkv[:, 4:]), want) and torch.equal(qkv[:, 4:], want)  # rows that interleave
    h, lens = ops.default_handle(), i32([3, 4])
    acc = torch.zeros(2, 2, 16, device="cuda")
    cfg = _lib.CacheAttnConfig(4, 2, 64, 16, 16, 0, 0.0)
    x = rnd(18, 2, 1, 4, 64)
    for out, a in [(ck, acc), (cv, acc), (x, acc), (acc, acc), (rnd(19, 2, 1, 4, 64), ck), (rnd(19, 2, 1, 4, 64), cv)]:
        refused(lambda: h.check(h.lib.fm_attention_scored(h.h, _lib.C.byref(cfg), x.data_ptr(), ck.data_ptr(), cv.data_ptr(),
                                                          lens.data_ptr(), 2, 1, a.data_ptr(), out.data_ptr())), _lib.FM_EINVAL)
    refused(lambda: h.check(h.lib.fm_attention_prefix(h.h, _lib.C.byref(cfg), x.data_ptr(), ck.data_ptr(), cv.data_ptr(), 16,
                                                      None, None, None, 2, 1, cv.data_ptr())), _lib.FM_EINVAL)
    refused(lambda: ops.cache_evict(ck, ck, acc, lens, 3), _lib.FM_EINVAL)
    new = rnd(20, 2, 2, 16, 64)
    refused(lambda: ops.cache_evict(ck, cv, acc, lens, 3, out=(new, new, torch.zeros_like(acc), None)), _lib.FM_EINVAL)


def test_numbers_beyond_their_c_types_are_refused():
    from flashmlx_b200 import ops
    ck, cv, acc, lens = rnd(21, 2, 2, 16, 64), rnd(22, 2, 2, 16, 64), torch.zeros(2, 2, 16, device="cuda"), i32([9, 16])
    for call in [
        lambda: ops.cache_evict(ck, cv, acc, lens, 2 ** 32 + 5), lambda: ops.cache_evict(ck, cv, acc, lens, 5, recent=2 ** 32),
        lambda: ops.cache_evict(ck, cv, acc, lens, 5, sinks=2 ** 32),
        lambda: ops.attention_prefix(rnd(23, 2, 1, 4, 64), None, None, ck, cv, lens, scale=1e-60),
        lambda: ops.attention_prefix(rnd(23, 2, 1, 4, 64), None, None, ck, cv, lens, scale=1e60),
    ]:
        refused(call)


# ------------------------------------------------------------------ rotary positions
YARN = {"type": "yarn", "factor": 4.0, "original_len": 4096, "beta_slow": 1.0, "beta_fast": 32.0}
BANDED = {"type": "banded", "factor": 8.0, "original_len": 8192, "low_freq": 1.0, "high_freq": 4.0}


@pytest.mark.parametrize("T,heads,d,rotary,traditional,scaling", [
    (1, 1, 8, None, False, None),
    (1, 36, 128, None, False, None),
    (5, 4, 64, 32, True, {"type": "linear", "factor": 4.0}),
    (3, 2, 64, 20, False, YARN),                       # half of 10: pair by pair
    (3, 3, 24, 6, True, {"type": "ntk", "factor": 2.0}),
    (7, 2, 128, 64, True, BANDED),
    (129, 5, 256, 2, False, None),
    (1300, 6, 64, None, False, YARN),                  # several tokens a block, a ragged last block
    (1301, 2, 128, 96, True, {"type": "yarn", "factor": 2.0, "original_len": 512, "beta_slow": 1.0, "beta_fast": 32.0,
                              "attn_factor": 1.25}),
])
def test_rope(T, heads, d, rotary, traditional, scaling):
    from flashmlx_b200 import ops
    x = rnd(10 + T, T, heads, d)
    g = torch.Generator().manual_seed(T)
    pos = torch.randint(-2000000, 2000000, (T,), generator=g, dtype=torch.int32)
    pos[0] = 2 ** 31 - 1
    if T > 2:
        pos[1], pos[2] = -2 ** 31, 0
    want, tol = R.rope(x, pos, 1e4, rotary, traditional, scaling)
    kw = dict(rotary_dim=rotary, traditional=traditional, scaling=scaling)
    y = ops.rope(x, pos.cuda(), 1e4, **kw)
    held(y, want, tol)
    # in place inside a wider row (a fused projection's), whose other columns stay
    wide = rnd(11, T, (heads + 2) * d)
    before = wide.clone()
    view = wide[:, d:(heads + 1) * d].view(T, heads, d)
    view.copy_(x)
    assert ops.rope(view, pos.cuda(), 1e4, out=view, **kw) is view
    assert torch.equal(view, y)
    assert torch.equal(wide[:, :d], before[:, :d]) and torch.equal(wide[:, (heads + 1) * d:], before[:, (heads + 1) * d:])


def test_rope_turns_back():
    """Negated positions undo a rotation but for the two roundings."""
    from flashmlx_b200 import ops
    x, pos = rnd(12, 40, 3, 128), torch.arange(1000, 1040, dtype=torch.int32, device="cuda")
    back = ops.rope(ops.rope(x, pos, 1e6), -pos, 1e6)
    f = x.double().cpu()
    size = f.abs() + torch.cat((f[..., 64:], f[..., :64]), -1).abs()
    held(back, f, size * (3 * R.U16))


def test_rope_no_tokens():
    from flashmlx_b200 import ops
    assert ops.rope(rnd(1, 0, 2, 64), i32([]), 1e4).shape == (0, 2, 64)


@pytest.mark.parametrize("B,L,nh,nkv,d,traditional,rotary", [
    (1, 1, 4, 4, 128, False, None), (3, 5, 4, 2, 64, True, 32), (2, 7, 6, 2, 40, False, 12), (2, 600, 2, 1, 64, False, None)])
def test_rope_append(B, L, nh, nkv, d, traditional, rotary):
    from flashmlx_b200 import ops
    M, T = L + 9, B * L
    qkv = rnd(20, T, nh + 2 * nkv, d)
    q, k, v = qkv[:, :nh], qkv[:, nh:nh + nkv], qkv[:, nh + nkv:]
    ck, cv = rnd(21, B, nkv, M, d), rnd(22, B, nkv, M, d)
    ck0, cv0 = ck.clone(), cv.clone()
    slots = torch.stack([torch.randperm(M, generator=torch.Generator().manual_seed(b))[:L] for b in range(B)]).int()
    slots[-1, L // 2] = -1  # a padding token
    pos = torch.arange(100, 100 + T, dtype=torch.int32)
    before = qkv.clone()
    got = ops.rope_append(q, k, v, pos.cuda(), slots.reshape(-1).cuda(), ck, cv, 1e6, traditional=traditional,
                          rotary_dim=rotary)
    assert torch.equal(qkv, before)
    held(got, *R.rope(q, pos, 1e6, rotary, traditional), what="q")
    rot = ops.rope(k, pos.cuda(), 1e6, rotary_dim=rotary, traditional=traditional)  # held to the formula above
    for t in range(T):
        s = int(slots.reshape(-1)[t])
        if s >= 0:
            ck0[t // L, :, s], cv0[t // L, :, s] = rot[t], v[t]
    assert torch.equal(ck, ck0) and torch.equal(cv, cv0)
    assert ops.rope_append(q, k, v, pos.cuda(), slots.reshape(-1).cuda(), ck, cv, 1e6, traditional=traditional,
                           rotary_dim=rotary, out=q) is q
    assert torch.equal(q, got)


def test_rope_append_reports_a_slot_past_the_cache():
    from flashmlx_b200 import _lib, ops
    ck, cv = rnd(23, 1, 2, 8, 64), rnd(24, 1, 2, 8, 64)
    k0, x = ck.clone(), rnd(25, 2, 2, 64)
    ops.rope_append(x, x, x, i32([0, 1]), i32([8, 3]), ck, cv, 1e4)
    with pytest.raises(_lib.FlashMoEError) as e:
        ops.synchronize()
    assert e.value.status == _lib.FM_EDEVICE
    k0[:, :, 3] = ck[:, :, 3]
    assert torch.equal(ck, k0) and torch.equal(cv[0, :, 3], x[1])


# ------------------------------------------------------------------ attention
def caches(seed, B, nkv, M, d, lens):
    """Random caches whose slots past each length are NaN (K) and infinite (V)."""
    ck, cv = rnd(seed, B, nkv, M, d), rnd(seed + 1, B, nkv, M, d)
    for b, n in enumerate(lens):
        ck[b, :, max(n, 0):] = float("nan")
        cv[b, :, max(n, 0):] = float("inf")
    return ck, cv


@pytest.mark.parametrize("B,L,nh,nkv,d,P,lens,M", [
    (1, 1, 1, 1, 64, 1, [0], 1),
    (1, 1, 4, 4, 128, 0, [1], 3),
    (3, 1, 4, 2, 64, 97, [1, 17, 41], 41),
    (2, 1, 32, 4, 128, 300, [0, 129], 130),
    (4, 3, 8, 2, 64, 63, [3, 2, 0, 70], 75),            # fewer slots than tokens: early ones see the prefix alone
    (3, 2, 6, 2, 128, 0, [1, 0, 33], 40),               # rows that see nothing
    (5, 1, 16, 16, 128, 129, [5, 128, 16, 127, 255], 256),
    (2, 17, 8, 2, 64, 40, [17, 64], 64),
    (1, 70, 6, 2, 128, 31, [200], 207),
    (40, 1, 8, 2, 64, 1000, list(range(0, 80, 2)), 80),
    (2, 1, 4, 2, 128, 5000, [7, 3], 9),
    (1, 300, 4, 1, 64, 10, [300], 300),
    (33, 5, 8, 2, 128, 517, [5 + 9 * (i % 7) for i in range(33)], 60),
    (3, 40, 8, 2, 64, 0, [10, 40, 0], 64),              # many rows that see nothing
    (2, 100, 8, 2, 128, 0, [7, 333], 340),
    (1, 129, 4, 4, 128, 0, [500], 512),                 # one head a kv head, a ragged second row tile
    (2, 50, 7, 1, 128, 0, [256, 50], 256),              # 350 rows in groups of 7
    (1, 9, 64, 1, 64, 1500, [9], 9),                    # 64 heads on one kv head
])
def test_attention_prefix(B, L, nh, nkv, d, P, lens, M):
    from flashmlx_b200 import ops
    q = rnd(30 + B + L, B, L, nh, d)
    ck, cv = caches(31, B, nkv, M, d, lens)
    pk = pv = None
    if P:
        pk, pv = rnd(33, nkv, P, d), rnd(34, nkv, P, d)
    out = ops.attention_prefix(q, pk, pv, ck, cv, i32(lens))
    want, tol, _, _ = R.attention(q, ck, cv, lens, pk, pv)
    held(out, want, tol)
    # q rows of a fused projection, the prefix in a longer buffer
    wide = rnd(35, B, L, nh + 2 * nkv, d)
    wide[:, :, :nh] = q
    long = [None, None]
    if P:
        long = [torch.full((nkv, P + 21, d), float("nan"), dtype=BF, device="cuda") for _ in range(2)]
        long[0][:, :P], long[1][:, :P] = pk, pv
    again = ops.attention_prefix(wide[:, :, :nh], long[0], long[1], ck, cv, i32(lens), prefix_len=P if P else None)
    assert torch.equal(again, out)


def test_attention_prefix_alone():
    from flashmlx_b200 import ops
    q, pk, pv = rnd(40, 9, 2, 8, 64), rnd(41, 4, 130, 64), rnd(42, 4, 130, 64)
    want, tol, _, _ = R.attention(q, None, None, None, pk, pv)
    held(ops.attention_prefix(q, pk, pv), want, tol)
    assert torch.equal(ops.attention_prefix(q, pk, pv, prefix_len=0), torch.zeros_like(q))


def test_attention_prefix_large_scores():
    """Scores of several hundred: the running maximum, not the exponent's range, carries them."""
    from flashmlx_b200 import ops
    q, lens = rnd(43, 2, 1, 4, 64, std=30.0), [200, 90]
    ck, cv = caches(44, 2, 2, 200, 64, lens)
    pk, pv = rnd(46, 2, 100, 64, std=10.0), rnd(47, 2, 100, 64)
    want, tol, _, _ = R.attention(q, ck, cv, lens, pk, pv)
    held(ops.attention_prefix(q, pk, pv, ck, cv, i32(lens)), want, tol)


@pytest.mark.parametrize("B,nh,nkv,d,P,own", [(40, 8, 2, 64, 900, 30), (33, 16, 2, 128, 700, 0), (20, 4, 1, 128, 1300, 77)])
def test_attention_prefix_rising_scores(B, nh, nkv, d, P, own):
    """Scores that keep rising along the keys, by several powers of two at every tile: the running
    reference moves again and again, in the first and the second half of a tile's keys."""
    from flashmlx_b200 import ops
    q = rnd(140, B, 1, nh, d).abs() * 2
    lens = [own] * B
    ck, cv = caches(141, B, nkv, max(own, 1), d, lens)
    pk, pv = rnd(142, nkv, P, d), rnd(143, nkv, P, d)
    ramp = torch.arange(P, device="cuda")[None, :, None] / 160.0 + torch.randint(0, 2, (nkv, P, 1), device="cuda",
                                                                             generator=torch.Generator("cuda").manual_seed(1)) * 0.3
    pk = (pk * 0.1 + ramp / d ** 0.5).to(BF)
    want, tol, _, _ = R.attention(q, ck, cv, lens, pk, pv)
    held(ops.attention_prefix(q, pk, pv, ck, cv, i32(lens)), want, tol)
    acc = torch.zeros(1, nkv, P, device="cuda")  # the same keys as one sequence's own, 17 tokens
    q1 = rnd(144, 1, 17, nh, d).abs() * 2
    want, tol, a, at = R.attention(q1, pk[None], pv[None], [P], acc=acc)
    held(ops.attention_scored(q1, pk[None].contiguous(), pv[None].contiguous(), i32([P]), acc), want, tol)
    held(acc, a, at)


@pytest.mark.parametrize("B,L,nh,nkv,d,P,lens,M", [
    (2, 4, 8, 2, 64, 40, [50, 128], 130),                # up to 64 rows to a key
    (3, 17, 2, 2, 128, 0, [64, 17, 5], 70),
    (2, 16, 8, 2, 128, 33, [333, 21], 340),
    (1, 70, 1, 1, 64, 0, [200], 200),                    # up to 128
    (3, 30, 8, 2, 128, 0, [300, 30, 128], 310),
    (2, 40, 8, 2, 128, 50, [300, 129], 300),             # up to 256
    (2, 300, 4, 2, 64, 100, [700, 320], 701),            # several row tiles
    (1, 600, 8, 1, 128, 0, [2000], 2000),
    (1, 515, 3, 3, 128, 0, [515], 530),
    (40, 150, 4, 2, 64, 0, [150 + 3 * i for i in range(40)], 300),
])
def test_attention_hides_values_that_are_not_finite(B, L, nh, nkv, d, P, lens, M):
    """Infinities and NaN in V reach the tokens that see their slot, in their column, and no other;
    NaN in the last token's K spoils that token alone."""
    from flashmlx_b200 import ops
    q = rnd(150 + L, B, L, nh, d)
    ck, cv = caches(151, B, nkv, M, d, lens)
    pk = pv = None
    if P:
        pk, pv = rnd(153, nkv, P, d), rnd(154, nkv, P, d)
    finite = cv.clone()
    group, extra = nh // nkv, torch.zeros(B, L, nh, d, dtype=torch.float64)
    values = [float("nan"), float("inf"), -float("inf")]
    for b, n in enumerate(lens):
        for i, slot in enumerate(sorted({n - 1, n - 2, n - L // 2, n - 2 * L // 3, n - L + 1, n - L, n - L - 1})):
            if not 0 <= slot < n:
                continue
            for h in range(nkv):
                for col in {(5 * i + 3 * h) % d, (d // 2 + 7 * i) % d, d - 1 - i}:
                    x = values[(i + h + col) % 3]
                    cv[b, h, slot, col], finite[b, h, slot, col] = x, 0.0
                    extra[b, max(slot - (n - L), 0):, h * group:(h + 1) * group, col] += x
    acc = torch.zeros(B, nkv, M, device="cuda")
    want, tol, a, at = R.attention(q, ck, finite, lens, pk, pv, acc=acc if not P else None)
    spoiled = ~torch.isfinite(extra)

    def check(out, keep=slice(None)):
        out = out.cpu().double()
        assert torch.equal(out[:, keep][spoiled[:, keep]].nan_to_num(nan=7.0), extra[:, keep][spoiled[:, keep]].nan_to_num(nan=7.0))
        held(torch.where(spoiled, want, out)[:, keep], want[:, keep], tol[:, keep])

    check(ops.attention_prefix(q, pk, pv, ck, cv, i32(lens)))
    if not P:
        check(ops.attention_scored(q, ck, cv, i32(lens), acc))
        held(acc, a, at)
    for b, n in enumerate(lens):  # stale memory where a padding token was not written
        ck[b, :, n - 1] = float("nan")
    out = ops.attention_prefix(q, pk, pv, ck, cv, i32(lens))
    check(out, slice(0, L - 1))
    assert torch.isnan(out[:, L - 1]).all()


@pytest.mark.parametrize("scale", [0.25, -0.1])
def test_attention_scale(scale):
    from flashmlx_b200 import ops
    q, lens = rnd(48, 2, 3, 4, 64), [30, 5]
    ck, cv = caches(49, 2, 2, 33, 64, lens)
    acc = torch.zeros(2, 2, 33, device="cuda")
    want, tol, a, at = R.attention(q, ck, cv, lens, acc=acc, scale=scale)
    held(ops.attention_scored(q, ck, cv, i32(lens), acc, scale=scale), want, tol)
    held(acc, a, at)


@pytest.mark.parametrize("B,L,nh,nkv,d,lens,M", [
    (1, 1, 1, 1, 64, [1], 1),
    (2, 1, 4, 4, 128, [0, 37], 40),
    (3, 1, 32, 4, 128, [1, 700, 129], 700),
    (2, 4, 8, 2, 64, [2, 100], 101),
    (1, 130, 8, 2, 64, [130], 131),
    (2, 200, 6, 2, 128, [333, 200], 340),
    (1, 513, 4, 1, 64, [600], 600),
    (3, 60, 8, 2, 128, [20, 60, 0], 64),
    (2, 37, 7, 1, 64, [300, 129], 300),
    (1, 1100, 8, 2, 128, [1100], 1100),
    (1, 300, 2, 2, 128, [1000], 1024),
    (17, 1, 16, 16, 64, [3 * i for i in range(17)], 64),
    (3, 2, 4, 2, 64, [1025, 7, 2050], 2051),             # an odd leading size, several blocks of slots
])
def test_attention_scored(B, L, nh, nkv, d, lens, M):
    from flashmlx_b200 import ops
    q = rnd(50 + L, B, L, nh, d)
    ck, cv = caches(51, B, nkv, M, d, lens)
    acc = torch.rand(B, nkv, M, generator=torch.Generator().manual_seed(5)).cuda()
    first = acc.clone()
    want, tol, a, at = R.attention(q, ck, cv, lens, acc=acc)
    out = ops.attention_scored(q, ck, cv, i32(lens), acc)
    held(out, want, tol, "out")
    held(acc, a, at, "acc")
    for b, n in enumerate(lens):
        assert torch.equal(acc[b, :, n:], first[b, :, n:])
    twice = first.clone()  # the same sums in the same order every time
    assert torch.equal(ops.attention_scored(q, ck, cv, i32(lens), twice), out) and torch.equal(twice, acc)


def test_lengths_out_of_range_are_reported():
    from flashmlx_b200 import _lib, ops
    q = rnd(60, 3, 1, 4, 64)
    ck, cv = rnd(61, 3, 2, 16, 64), rnd(62, 3, 2, 16, 64)
    acc = torch.zeros(3, 2, 16, device="cuda")
    lens = [17, 9, -1]
    out = ops.attention_scored(q, ck, cv, i32(lens), acc)
    with pytest.raises(_lib.FlashMoEError) as e:
        ops.synchronize()
    assert e.value.status == _lib.FM_EDEVICE
    want, tol, a, at = R.attention(q, ck, cv, [0, 9, 0], acc=torch.zeros(3, 2, 16))
    held(out, want, tol)
    held(acc, a, at)


def test_attention_far_into_a_large_cache():
    """Element offsets past 2^31."""
    from flashmlx_b200 import ops
    B, nkv, M, d = 34, 8, 65536, 128
    ck = torch.empty(B, nkv, M, d, dtype=BF, device="cuda")
    cv = torch.empty_like(ck)
    lens = [0] * B
    lens[-1] = 200
    ck[-1, :, :200], cv[-1, :, :200] = rnd(63, nkv, 200, d), rnd(64, nkv, 200, d)
    q = rnd(65, B, 1, 8, d)
    out = ops.attention_prefix(q, None, None, ck, cv, i32(lens))
    want, tol, _, _ = R.attention(q[-1:], ck[-1:, :, :200], cv[-1:, :, :200], [200])
    held(out[-1:], want, tol)
    assert not out[:-1].any()
    acc = torch.rand(B, nkv, M, device="cuda")
    acc[-1, :, 50] = 9.0
    k50 = ck[-1, :, 50].clone()
    ops.cache_evict(ck, cv, acc, i32(lens), 10)
    assert (ck[-1, :, :10] == k50[:, None]).all(-1).any(-1).all()


# ------------------------------------------------------------------ eviction
@pytest.mark.parametrize("B,nkv,d,M,lens,budget,sinks,recent,weights", [
    (1, 1, 64, 1, [1], 1, 0, 0, "rand"),
    (2, 2, 64, 20, [20, 3], 7, 0, 0, "rand"),
    (2, 2, 128, 41, [0, 41], 40, 4, 8, "rand"),
    (3, 1, 64, 70, [70, 64, 33], 32, 2, 30, "ties"),
    (2, 2, 8, 33, [33, 20], 5, 0, 0, "zeros"),
    (2, 3, 40, 50, [50, 49], 16, 1, 3, "odd"),          # NaN, infinities, negative zeros
    (1, 2, 256, 3000, [2999], 1500, 4, 100, "rand"),
    (2, 2, 64, 5000, [5000, 1025], 1024, 0, 512, "ties"),
    (1, 1, 64, 100, [100], 200, 0, 0, "rand"),           # nothing to evict
    (1, 1, 8, 50000, [49990], 20001, 3, 77, "rand"),     # more keys than shared memory holds
    (1, 2, 8, 4096, [4096], 4095, 0, 4095, "ties"),      # one too many, nearly all protected
    (2, 3, 16, 16384, [16384, 9001], 2048, 4, 512, "odd"),  # heads that several CTAs share
    (3, 1, 8, 9000, [100, 8999, 33], 50, 0, 0, "zeros"),
    (1, 1, 8, 200000, [199999], 70001, 3, 77, "ties"),
    (1, 1, 8, 100000, [100000], 3, 1, 2, "rand"),
    (5, 8, 8, 16500, [16500, 4097, 0, 2049, 1], 2048, 10, 0, "rand"),
])
@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("given", [True, False])
def test_cache_evict(B, nkv, d, M, lens, budget, sinks, recent, weights, in_place, given):
    from flashmlx_b200 import ops
    ck, cv = rnd(70, B, nkv, M, d), rnd(71, B, nkv, M, d)
    g = torch.Generator().manual_seed(M + budget)
    acc = torch.rand(B, nkv, M, generator=g)
    if weights == "ties":
        acc = (acc * 4).floor()
    elif weights == "zeros":
        acc.zero_()
    elif weights == "odd":
        acc[..., ::3], acc[..., 1::7], acc[..., 2::11], acc[..., 5::9] = float("nan"), float("inf"), -float("inf"), -0.0
        acc[..., 6::9] = 0.0
    pos = None
    if given:  # positions in an order of their own, as after earlier evictions
        pos = torch.stack([torch.randperm(3 * M, generator=g)[:M] for _ in range(B * nkv)]).view(B, nkv, M).int()
    host = [ck.cpu(), cv.cpu(), acc.clone(), pos.clone() if given else None]
    n = M if in_place else min(budget, M) + 3
    to = host if in_place else [torch.zeros(B, nkv, n, d, dtype=BF), torch.zeros(B, nkv, n, d, dtype=BF),
                                torch.zeros(B, nkv, n), torch.zeros(B, nkv, n, dtype=torch.int32)]
    dev = [ck, cv, acc.cuda(), pos.cuda() if given else None]
    out = dev if in_place else [t.cuda() for t in to]
    source = [t.clone() if t is not None else None for t in host]
    want = R.evict(host[0], host[1], host[2], host[3], lens, budget, sinks, recent, to)
    lens_t = i32(lens)
    got = ops.cache_evict(dev[0], dev[1], dev[2], lens_t, budget, sinks=sinks, recent=recent, positions=dev[3],
                          out=None if in_place else tuple(out), lens_out=lens_t if in_place else None)
    assert got.tolist() == want
    for a, b in zip(out, to):
        if b is not None:
            assert torch.equal(a.cpu().nan_to_num(nan=-7.0), b.nan_to_num(nan=-7.0))
    if not in_place:
        for a, b in zip(dev, source):
            if b is not None:
                assert torch.equal(a.cpu().nan_to_num(nan=-7.0), b.nan_to_num(nan=-7.0))
        assert lens_t.tolist() == lens


@pytest.mark.parametrize("B,nkv,M,lens,budget", [(2, 2, 16400, [16400, 16395], 16390), (40, 1, 16384, [16384] * 39 + [5], 16383),
                                                 (3, 2, 60, [60, 3, 41], 40)])
def test_evict_a_few_slots_into_new_lengths(B, nkv, M, lens, budget):
    """In place with lens_out apart from lens: a few moves, made by the kernel that selects."""
    from flashmlx_b200 import ops
    dev = [rnd(170, B, nkv, M, 64), rnd(171, B, nkv, M, 64), torch.rand(B, nkv, M, generator=torch.Generator().manual_seed(3)).cuda()]
    host = [t.cpu().clone() for t in dev]
    want = R.evict(*host, None, lens, budget, 4, 16, [*host, None])
    assert ops.cache_evict(*dev, i32(lens), budget, sinks=4, recent=16).tolist() == want
    for x, y in zip(dev, host):
        assert torch.equal(x.cpu(), y)


@pytest.mark.parametrize("in_place", [True, False])
def test_a_captured_eviction_follows_its_inputs(in_place):
    """Heads that a cluster shares, in a graph replayed over other lengths and weights."""
    from flashmlx_b200 import ops
    B, nkv, M, budget, d = 2, 2, 16384, 700, 8
    h = ops.Handle()
    k, v = rnd(180, B, nkv, M, d), rnd(181, B, nkv, M, d)
    acc, lens = torch.zeros(B, nkv, M, device="cuda"), i32([M, M])
    dev = [k.clone(), v.clone(), acc.clone()]
    out = dev if in_place else [torch.zeros(B, nkv, budget, d, dtype=BF, device="cuda") for _ in range(2)] + \
        [torch.zeros(B, nkv, budget, device="cuda")]

    def step():
        for x, y in zip(dev, (k, v, acc)):
            x.copy_(y)
        return ops.cache_evict(*dev, lens, budget, sinks=4, recent=50, out=None if in_place else (*out, None), handle=h)

    step()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        n = step()
    for i, now in enumerate([[M, 9000], [3, 16001], [701, 0]]):
        acc.copy_(torch.rand(B, nkv, M, generator=torch.Generator().manual_seed(i)))
        lens.copy_(i32(now))
        for x in out if not in_place else []:
            x.zero_()
        g.replay()
        torch.cuda.synchronize()
        host = [x.cpu().clone() for x in (k, v, acc)]
        to = host if in_place else [torch.zeros(x.shape, dtype=x.dtype) for x in out]
        assert n.tolist() == R.evict(*host, None, now, budget, 4, 50, [*to, None])
        for x, y in zip(out, to):
            assert torch.equal(x.cpu(), y), f"replay {i}"
    h.sync()


def test_evict_reports_a_length_past_the_cache():
    from flashmlx_b200 import _lib, ops
    ck, cv, acc = rnd(72, 2, 1, 16, 64), rnd(73, 2, 1, 16, 64), torch.rand(2, 1, 16, device="cuda")
    k0 = ck.clone()
    got = ops.cache_evict(ck, cv, acc, i32([17, 16]), 8)
    with pytest.raises(_lib.FlashMoEError) as e:
        ops.synchronize()
    assert e.value.status == _lib.FM_EDEVICE
    assert got.tolist() == [0, 8] and torch.equal(ck[0], k0[0])


# ------------------------------------------------------------------ together
def test_a_conversation_that_evicts():
    """Steps as a server makes them: append, attend and weigh, evict when over the budget; every
    output, weight and cache against the plain forms carried along in 64 bits (the caches' bf16
    rows are taken over, so that each step's error is its own)."""
    from flashmlx_b200 import ops
    B, nh, nkv, d, M, budget, sinks, recent, theta = 3, 4, 2, 64, 40, 32, 2, 6, 1e6
    ck, cv = (torch.full((B, nkv, M, d), float("nan"), dtype=BF, device="cuda") for _ in range(2))
    acc = torch.zeros(B, nkv, M, device="cuda")
    positions = torch.zeros(B, nkv, M, dtype=torch.int32, device="cuda")
    lens, seen = [0] * B, [0] * B
    for step, new in enumerate([20, 1, 1, 9, 1, 1, 1, 7, 1, 1]):
        qkv = rnd(80 + step, B * new, nh + 2 * nkv, d)
        slots = torch.tensor([[lens[b] + i for i in range(new)] for b in range(B)], dtype=torch.int32)
        pos = torch.tensor([[seen[b] + 10 * b + i for i in range(new)] for b in range(B)], dtype=torch.int32)
        q = ops.rope_append(qkv[:, :nh], qkv[:, nh:nh + nkv], qkv[:, nh + nkv:], pos.view(-1).cuda(),
                            slots.view(-1).cuda(), ck, cv, theta)
        for b in range(B):
            positions[b, :, lens[b]:lens[b] + new] = pos[b].cuda()
            acc[b, :, lens[b]:lens[b] + new] = 0
            lens[b] += new
            seen[b] += new
        before = acc.clone()
        q = q.view(B, new, nh, d)
        want, tol, a, at = R.attention(q, ck, cv, lens, acc=before)
        out = ops.attention_scored(q, ck, cv, i32(lens), acc)
        held(out, want, tol, f"step {step}")
        held(acc, a, at, f"step {step} acc")
        host = [t.cpu().clone() for t in (ck, cv, acc, positions)]
        to = R.evict(*host, lens, budget, sinks, recent, host)
        lens_t = i32(lens)
        ops.cache_evict(ck, cv, acc, lens_t, budget, sinks=sinks, recent=recent, positions=positions, lens_out=lens_t)
        assert lens_t.tolist() == to
        lens = to
        for x, y in zip((ck, cv, acc, positions), host):
            assert torch.equal(x.cpu().nan_to_num(nan=-7.0), y.nan_to_num(nan=-7.0)), f"step {step}"


def test_a_captured_step_follows_its_lengths():
    """One graph of append + attention, replayed as the caches grow; a call that would grow the
    workspace inside a capture is refused and the capture goes on."""
    from flashmlx_b200 import _lib, ops
    B, nh, nkv, d, M, P = 4, 8, 2, 64, 96, 50
    h = ops.Handle()
    pk, pv = rnd(90, nkv, P, d), rnd(91, nkv, P, d)
    ck, cv = (torch.full((B, nkv, M, d), float("nan"), dtype=BF, device="cuda") for _ in range(2))
    start = [0, 7, 30, 64]
    for b, n in enumerate(start):
        ck[b, :, :n], cv[b, :, :n] = rnd(92 + b, nkv, n, d), rnd(96 + b, nkv, n, d)
    qkv = torch.zeros(B, nh + 2 * nkv, d, dtype=BF, device="cuda")
    slots, lens = i32(start), i32([n + 1 for n in start])

    def step():
        q = ops.rope_append(qkv[:, :nh], qkv[:, nh:nh + nkv], qkv[:, nh + nkv:], slots, slots, ck, cv, 1e6, handle=h)
        return ops.attention_prefix(q.view(B, 1, nh, d), pk, pv, ck, cv, lens, handle=h)

    keep = ck.clone(), cv.clone()  # the step before the capture sizes the workspace
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    ck.copy_(keep[0]), cv.copy_(keep[1])
    many = rnd(99, 4000, 1, nh, d)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
        with pytest.raises(_lib.FlashMoEError) as e:
            ops.attention_prefix(many, pk, pv, handle=h)
        assert e.value.status == _lib.FM_EINVAL
    big = ops.attention_prefix(many, pk, pv, handle=h)  # now it grows; the graph's block stays
    want, tol, _, _ = R.attention(many[:3], None, None, None, pk, pv)
    held(big[:3], want, tol)
    for i in range(3):
        qkv.copy_(rnd(100 + i, B, nh + 2 * nkv, d))
        g.replay()
        torch.cuda.synchronize()
        q = ops.rope(qkv[:, :nh], slots, 1e6)  # held to the formula in test_rope
        n = [s + 1 + i for s in start]
        assert not torch.isnan(ck[0, :, :n[0]]).any()
        want, tol, _, _ = R.attention(q.view(B, 1, nh, d), ck, cv, n, pk, pv)
        held(out, want, tol, f"replay {i}")
        slots += 1
        lens += 1
    h.sync()


def test_a_captured_step_between_copies_and_forks():
    """The calls begin while what is in front of them ends; a clear, a copy or another stream's
    kernel in front is waited for, in a graph and out of it."""
    from flashmlx_b200 import ops
    B, nh, nkv, d, M = 3, 32, 4, 128, 4000
    h = ops.Handle()
    ck, cv, k2, v2 = (torch.zeros(B, nkv, M, d, dtype=BF, device="cuda") for _ in range(4))
    src_k, src_v, q = rnd(160, B, nkv, M, d), rnd(161, B, nkv, M, d), rnd(162, B, 6, nh, d)
    lens, want_lens = torch.zeros(B, dtype=torch.int32, device="cuda"), i32([4000, 17, 2100])
    acc, a2 = (torch.ones(B, nkv, M, device="cuda") for _ in range(2))
    other = torch.cuda.Stream()

    def step():
        here = torch.cuda.current_stream()
        other.wait_stream(here)
        with torch.cuda.stream(other):
            cv.copy_(src_v)
        ck.copy_(src_k)
        acc.zero_()
        lens.copy_(want_lens)
        here.wait_stream(other)
        out = ops.attention_scored(q, ck, cv, lens, acc, handle=h)
        a2.copy_(acc)
        n = ops.cache_evict(ck, cv, acc, lens, 1000, sinks=4, recent=100, handle=h)
        k2.copy_(ck), v2.copy_(cv)
        ck.zero_(), cv.zero_()
        return out, n

    want, tol, a, at = R.attention(q, src_k, src_v, want_lens.tolist(), acc=torch.zeros_like(acc))
    runs = []

    def check(out, n):
        torch.cuda.synchronize()
        held(out, want, tol)
        held(a2, a, at)
        assert n.tolist() == [1000, 17, 1000]
        runs.append([t.clone() for t in (out, a2, k2, v2, acc)])
        assert all(torch.equal(x, y) for x, y in zip(runs[0], runs[-1]))

    check(*step())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out, n = step()
    for _ in range(3):
        for t in (lens, acc, k2, v2, a2, out):
            t.zero_()
        g.replay()
        check(out, n)
    h.sync()


@pytest.mark.parametrize("nh,nkv,d,M,P,B,L", [(32, 4, 128, 700, 300, 9, 40), (4, 4, 64, 130, 0, 33, 3), (8, 1, 64, 2000, 5000, 1, 1)])
def test_reserved_calls_do_not_allocate(nh, nkv, d, M, P, B, L):
    """After fm_serve_reserve no call of up to its sizes grows the workspace."""
    from flashmlx_b200 import _lib, ops
    h = ops.Handle()
    cfg = _lib.CacheAttnConfig(nh, nkv, d, M, P, 0, 0.0)
    h.check(h.lib.fm_serve_reserve(h.h, _lib.C.byref(cfg), B, L))
    size = h.workspace_bytes()
    ck, cv = rnd(120, B, nkv, M, d), rnd(121, B, nkv, M, d)
    acc = torch.zeros(B, nkv, M, device="cuda")
    pk = rnd(122, nkv, P, d) if P else None
    for b in sorted({1, min(2, B), B // 2, B} - {0}):
        for n in sorted({1, min(2, L), L // 2, L} - {0}):
            q, lens = rnd(123, b, n, nh, d), i32([M] * b)
            ops.attention_prefix(q, pk, pk, ck[:b], cv[:b], lens, handle=h)
            ops.attention_scored(q, ck[:b], cv[:b], lens, acc[:b], handle=h)
    if P:
        ops.attention_prefix(rnd(124, B, L, nh, d), pk, pk, handle=h)
    ops.cache_evict(ck, cv, acc, i32([M] * B), M - 1, handle=h)
    h.sync()
    assert h.workspace_bytes() == size


def test_negative_positions_and_their_window():
    """recent counts from the newest position, whatever its sign; at the type's lowest value too."""
    from flashmlx_b200 import ops
    low = -2 ** 31
    pos = torch.tensor([low, low + 1, low + 2, low + 3, low + 4], dtype=torch.int32).view(1, 1, 5)
    ck, cv, acc = rnd(130, 1, 1, 5, 64), rnd(131, 1, 1, 5, 64), torch.tensor([5.0, 4, 3, 2, 1]).view(1, 1, 5)
    host = [ck.cpu().clone(), cv.cpu().clone(), acc.clone(), pos.clone()]
    R.evict(host[0], host[1], host[2], host[3], [5], 4, 0, 4, host)
    dev = [ck, cv, acc.cuda(), pos.cuda()]
    ops.cache_evict(dev[0], dev[1], dev[2], i32([5]), 4, recent=4, positions=dev[3])
    # (every position is protected: all lie below `sinks` = 0)
    for x, y in zip(dev, host):
        assert torch.equal(x.cpu(), y)


def test_two_streams_with_their_own_handles():
    from flashmlx_b200 import ops
    q, lens = rnd(110, 4, 1, 8, 128), [300, 20, 150, 77]
    ck, cv = caches(111, 4, 2, 300, 128, lens)
    one = ops.attention_prefix(q, None, None, ck, cv, i32(lens))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    handles = [ops.Handle() for _ in range(2)]
    n = i32(lens)
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        for s, h in zip(streams, handles):
            with torch.cuda.stream(s):
                got.append(ops.attention_prefix(q, None, None, ck, cv, n, handle=h))
    torch.cuda.synchronize()
    assert all(torch.equal(x, one) for x in got)


def test_the_first_report_outlasts_the_default_streams_work():
    """A handle's first serving call sets up its error word: on the call's stream, so that work queued on
    the default stream, which does not order other streams, cannot delay it past the report."""
    from flashmlx_b200 import _lib, ops
    h, side = ops.Handle(), torch.cuda.Stream()
    ck, cv, x, out = rnd(23, 1, 2, 8, 64), rnd(24, 1, 2, 8, 64), rnd(25, 2, 2, 64), rnd(26, 2, 2, 64)
    at, slots = i32([0, 1]), i32([8, 3])
    ops.rope_append(x, x, x, at, at, ck, cv, 1e4, out=out)  # the kernel is loaded
    torch.cuda.synchronize()
    torch.cuda._sleep(400_000_000)  # 0.2 s of the default stream
    with torch.cuda.stream(side):
        ops.rope_append(x, x, x, at, slots, ck, cv, 1e4, out=out, handle=h)
    with pytest.raises(_lib.FlashMoEError) as e:
        h.sync()
    assert e.value.status == _lib.FM_EDEVICE
    h.sync()  # reported once


def test_streams_that_share_a_handle_take_turns():
    """Without a handle given, calls on two streams share the default handle's workspace: the later
    call waits for the earlier one, whatever held that up."""
    from flashmlx_b200 import ops
    lens = [3000, 500, 2100, 77]
    n = i32(lens)
    data = []
    for i in range(2):
        q, acc = rnd(190 + i, 4, 6, 8, 128), torch.rand(4, 2, 3000, generator=torch.Generator().manual_seed(i)).cuda()
        data.append((q, *caches(192 + 2 * i, 4, 2, 3000, 128, lens), acc))

    def work(q, ck, cv, acc):
        ck, cv, acc = ck.clone(), cv.clone(), acc.clone()
        out = ops.attention_scored(q, ck, cv, n, acc)
        weights = acc.clone()
        new = ops.cache_evict(ck, cv, acc, n, 1500, sinks=4, recent=64)
        return [out, weights, ck, cv, acc, new]

    want = [work(*d) for d in data]
    ops.synchronize()
    streams, ends, got = [torch.cuda.Stream() for _ in range(2)], [], []
    for i in range(6):
        with torch.cuda.stream(streams[i % 2]):
            if i == 0:
                torch.cuda._sleep(400_000_000)  # 0.2 s
            got.append(work(*data[i % 2]))
            ends.append(torch.cuda.Event())
            ends[-1].record()
    assert not ends[1].query()  # behind the first stream's sleep
    ops.synchronize()
    assert all(e.query() for e in ends)
    for i, g in enumerate(got):
        for x, y in zip(g, want[i % 2]):
            assert torch.equal(x.nan_to_num(nan=-7.0), y.nan_to_num(nan=-7.0)), i


def test_a_captured_call_on_its_own_stream_between_eager_ones():
    """The default handle: eager calls before, in between (on another stream) and after a capture, whose
    own calls wait for nothing."""
    from flashmlx_b200 import _lib, ops
    lens = [300, 20, 150]
    q, (ck, cv), n = rnd(200, 3, 1, 8, 64), caches(201, 3, 2, 300, 64, lens), i32(lens)
    want = ops.attention_prefix(q, None, None, ck, cv, n)
    side, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    between, h, cfg = torch.zeros_like(q), ops.default_handle(), _lib.CacheAttnConfig(8, 2, 64, 300, 0, 0, 0.0)
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        out = ops.attention_prefix(q, None, None, ck, cv, n)
        with torch.cuda.stream(side):
            h.bind_current()  # (torch allocates on no other stream during a capture)
            h.check(h.lib.fm_attention_prefix(h.h, _lib.C.byref(cfg), q.data_ptr(), None, None, 0, ck.data_ptr(), cv.data_ptr(),
                                              n.data_ptr(), 3, 1, between.data_ptr()))
        again = ops.attention_prefix(q, None, None, ck, cv, n)
    after = ops.attention_prefix(q, None, None, ck, cv, n)
    ops.synchronize()
    assert torch.equal(after, want)
    for t in (out, again):
        t.zero_()
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want) and torch.equal(again, want) and torch.equal(between, want)
    ops.synchronize()


@pytest.mark.parametrize("L", [1, 5, 40])
@pytest.mark.parametrize("P", [0, 33])
def test_caches_without_slots(L, P):
    """max_len 0: every token sees the prefix alone, or nothing; a length above it is reported."""
    from flashmlx_b200 import _lib, ops
    q, empty, lens = rnd(210, 3, L, 8, 64), torch.empty(3, 2, 0, 64, dtype=BF, device="cuda"), i32([0, 0, 0])
    pk, pv = (rnd(211, 2, P, 64), rnd(212, 2, P, 64)) if P else (None, None)
    out = ops.attention_prefix(q, pk, pv, empty, empty, lens)
    assert torch.equal(out, ops.attention_prefix(q, pk, pv) if P else torch.zeros_like(q))
    if not P:
        acc = torch.empty(3, 2, 0, device="cuda")
        assert torch.equal(ops.attention_scored(q, empty, empty, lens, acc), torch.zeros_like(q))
    ops.synchronize()
    assert torch.equal(ops.attention_prefix(q, pk, pv, empty, empty, i32([0, 1, 0])), out)
    with pytest.raises(_lib.FlashMoEError) as e:
        ops.synchronize()
    assert e.value.status == _lib.FM_EDEVICE


@pytest.mark.parametrize("B,L,nh,nkv,d,lens", [
    (2, 40, 6, 2, 64, [300, 129]), (1, 50, 7, 1, 128, [200]), (1, 30, 65, 1, 64, [150]), (1, 3, 3, 1, 64, [90]),
    (2, 64, 8, 2, 128, [128, 260])])
def test_slots_of_minus_infinite_score_weigh_nothing(B, L, nh, nkv, d, lens):
    """A key of -infinity in one column scores -infinity with queries that are positive there: the call is as
    without the slot, whose weight stays (groups that do not fill a tile of 128 rows among them)."""
    from flashmlx_b200 import ops
    q, M, at = rnd(220 + L, B, L, nh, d).abs() + 0.125, max(lens) + 1, 20
    ck, cv = caches(221, B, nkv, M, d, lens)
    ck[:, :, at, 3] = -float("inf")
    acc = torch.rand(B, nkv, M, generator=torch.Generator().manual_seed(9)).cuda()
    first = acc.clone()
    keep = [i for i in range(M) if i != at]
    want, tol, a, at_tol = R.attention(q, ck[:, :, keep], cv[:, :, keep], [n - 1 for n in lens], acc=acc[:, :, keep])
    out = ops.attention_scored(q, ck, cv, i32(lens), acc)
    held(out, want, tol, "out")
    held(acc[:, :, keep], a, at_tol, "acc")
    assert torch.equal(acc[:, :, at], first[:, :, at])


@pytest.mark.parametrize("B,L,nh,nkv,d,lens", [
    (2, 4, 8, 2, 64, [100, 37]), (1, 2, 4, 4, 128, [700]), (2, 40, 8, 2, 64, [300, 129]), (1, 200, 6, 2, 128, [260])])
def test_a_token_of_nan_weighs_only_on_slots_that_it_sees(B, L, nh, nkv, d, lens):
    from flashmlx_b200 import ops
    M = max(lens)
    q = rnd(230 + L, B, L, nh, d)
    ck, cv = caches(231, B, nkv, M, d, lens)
    clean, acc = q.clone(), torch.zeros(B, nkv, M, device="cuda")
    q[0, 0, 0, 5], clean[0, 0, 0, 5] = float("nan"), 0.0
    want, tol, a, at = R.attention(clean, ck, cv, lens, acc=acc)
    out = ops.attention_scored(q, ck, cv, i32(lens), acc)
    assert torch.isnan(out[0, 0, 0]).all()
    out[0, 0, 0] = want[0, 0, 0].to(BF).cuda()
    held(out, want, tol, "out")
    seen = lens[0] - L + 1  # slots that the first token sees
    assert torch.isnan(acc[0, 0, :seen]).all()
    acc[0, 0, :seen] = a[0, 0, :seen].float().cuda()
    held(acc, a, at, "acc")


def test_a_capture_right_after_the_reservation():
    """fm_serve_reserve is enough: the handle's first calls may be captured ones."""
    from flashmlx_b200 import _lib, ops
    B, L, nh, nkv, d, M, P, lens = 3, 40, 8, 2, 128, 600, 200, [600, 41, 333]
    h, cfg = ops.Handle(), _lib.CacheAttnConfig(8, 2, 128, 600, 200, 0, 0.0)
    q, (ck, cv), n = rnd(240, B, L, nh, d), caches(241, B, nkv, M, d, lens), i32(lens)
    pk, pv, acc = rnd(243, nkv, P, d), rnd(244, nkv, P, d), torch.zeros(B, nkv, M, device="cuda")
    one, at = q[:, :1].contiguous(), torch.arange(B, dtype=torch.int32, device="cuda")
    h.check(h.lib.fm_serve_reserve(h.h, _lib.C.byref(cfg), B, L))

    def step(handle):
        r = ops.rope(one[:, 0], at, 1e4, handle=handle)
        outs = [r, ops.attention_prefix(q, pk, pv, ck, cv, n, handle=handle), ops.attention_scored(q, ck, cv, n, acc, handle=handle),
                ops.attention_scored(one, ck, cv, n, acc, handle=handle), ops.attention_prefix(one, pk, pv, ck, cv, n, handle=handle)]
        a = acc.clone()
        k, v = ck.clone(), cv.clone()
        return outs + [a, ops.cache_evict(k, v, a, n, 300, sinks=2, recent=20, handle=handle), k, v]

    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step(h)
    acc.zero_()
    g.replay()
    torch.cuda.synchronize()
    acc.zero_()
    for x, y in zip(got, step(None)):
        assert torch.equal(x.nan_to_num(nan=-7.0), y.nan_to_num(nan=-7.0))
    h.sync()


@pytest.mark.parametrize("M,lens,lo", [(40, [40, 33], -10), (300, [300, 290], 5), (3000, [2999, 1600], -1500), (17000, [17000, 9000], 100)])
@pytest.mark.parametrize("in_place", [True, False])
def test_the_recent_window_counts_from_the_newest_position(M, lens, lo, in_place):
    """Positions on both sides of 0, or all at or above the sinks, in a shuffled order; the recent slots are the
    lightest, so that only the window keeps them, and the sinks the next lightest."""
    from flashmlx_b200 import ops
    B, nkv, d, sinks, recent = len(lens), 2, 8, 6, 9
    g = torch.Generator().manual_seed(M)
    pos = torch.stack([torch.randperm(M, generator=g) + lo for _ in range(B * nkv)]).view(B, nkv, M).int()
    acc = 1.0 + torch.rand(B, nkv, M, generator=g)
    for b, n in enumerate(lens):
        for h in range(nkv):
            newest = int(pos[b, h, :n].max())
            acc[b, h, pos[b, h] > newest - recent] = 0.0
            acc[b, h, pos[b, h] < sinks] = 0.5
    budget = M - lo if lo < 0 else M // 2  # (below 0 all positions are the sinks')
    budget = min(budget, min(lens) - 1)
    dev = [rnd(250, B, nkv, M, d), rnd(251, B, nkv, M, d), acc.cuda(), pos.cuda()]
    host = [t.cpu().clone() for t in dev]
    out = dev if in_place else [torch.zeros(B, nkv, budget, *t.shape[3:], dtype=t.dtype, device="cuda") for t in dev]
    to = host if in_place else [torch.zeros(t.shape, dtype=t.dtype) for t in out]
    want = R.evict(*host, lens, budget, sinks, recent, to)
    got = ops.cache_evict(*dev[:3], i32(lens), budget, sinks=sinks, recent=recent, positions=dev[3],
                          out=None if in_place else tuple(out))
    assert got.tolist() == want
    for x, y in zip(out, to):
        assert torch.equal(x.cpu(), y)
    for b in range(B):  # the window's slots are among those that stay
        for h in range(nkv):
            held_at = set(to[3][b, h, :want[b]].tolist())
            top = int(pos[b, h, :lens[b]].max())
            here = set(pos[b, h, :lens[b]].tolist())
            assert {p for p in here if p > top - recent} <= held_at


@pytest.mark.parametrize("B,nkv,M,lens,budget,recent", [
    (2, 3, 18500, [18500, 9001], 2048, 512), (5, 8, 20000, [20000, 4097, 0, 2049, 1], 2048, 0),  # four, two CTAs a head
    (1, 1, 40000, [39990], 20001, 77), (38, 2, 18432, [18432 - 450 * i for i in range(38)], 2000, 99),  # one: too many heads
    (2, 2, 19000, [19000, 18890], 18875, 16), (17, 2, 18600, [18600] * 16 + [5], 18480, 16)])  # a few moves
@pytest.mark.parametrize("how", ["in place", "lens is lens_out", "elsewhere"])
def test_evict_long_caches(B, nkv, M, lens, budget, recent, how):
    from flashmlx_b200 import ops
    g, d = torch.Generator().manual_seed(M), 8
    acc = (torch.rand(B, nkv, M, generator=g) * 500).floor()
    pos = torch.stack([torch.randperm(3 * M, generator=g)[:M] for _ in range(B * nkv)]).view(B, nkv, M).int()
    dev = [rnd(260, B, nkv, M, d), rnd(261, B, nkv, M, d), acc.cuda(), pos.cuda()]
    host = [t.cpu().clone() for t in dev]
    inside = how != "elsewhere"
    out = dev if inside else [torch.zeros(B, nkv, budget, *t.shape[3:], dtype=t.dtype, device="cuda") for t in dev]
    to = host if inside else [torch.zeros(t.shape, dtype=t.dtype) for t in out]
    want = R.evict(*host, lens, budget, 4, recent, to)
    n = i32(lens)
    got = ops.cache_evict(*dev[:3], n, budget, sinks=4, recent=recent, positions=dev[3], out=None if inside else tuple(out),
                          lens_out=n if how == "lens is lens_out" else None)
    assert got.tolist() == want
    for x, y in zip(out, to):
        assert torch.equal(x.cpu(), y)


@pytest.mark.parametrize("slack", [1, 63, 64, 65, 127, 128, 129, 300])
@pytest.mark.parametrize("heads", [(3, 2), (40, 4)])
def test_evict_up_to_the_slack_of_a_cache(slack, heads):
    """Around the number of moves that the selecting kernel makes itself: all of them, and one."""
    from flashmlx_b200 import ops
    (B, nkv), budget, d = heads, 400, 16
    M = budget + slack
    lens = [budget + slack if i % 2 == 0 else budget + 1 for i in range(B)]
    acc = torch.rand(B, nkv, M, generator=torch.Generator().manual_seed(slack))
    acc[:, :, budget:] += 1.0  # the late slots stay, so that all of them move
    dev = [rnd(270, B, nkv, M, d), rnd(271, B, nkv, M, d), acc.cuda()]
    host = [t.cpu().clone() for t in dev]
    want = R.evict(*host, None, lens, budget, 2, 0, [*host, None])
    assert ops.cache_evict(*dev, i32(lens), budget, sinks=2).tolist() == want
    for x, y in zip(dev, host):
        assert torch.equal(x.cpu(), y)


@pytest.mark.parametrize("in_place", [True, False])
def test_a_captured_eviction_of_a_long_cache(in_place):
    """The cluster's kernel in a graph replayed over other lengths and weights."""
    from flashmlx_b200 import ops
    B, nkv, M, budget, d = 2, 2, 20000, 700, 8
    h = ops.Handle()
    k, v = rnd(280, B, nkv, M, d), rnd(281, B, nkv, M, d)
    acc, lens = torch.zeros(B, nkv, M, device="cuda"), i32([M, M])
    dev = [k.clone(), v.clone(), acc.clone()]
    out = dev if in_place else [torch.zeros(B, nkv, budget, d, dtype=BF, device="cuda") for _ in range(2)] + \
        [torch.zeros(B, nkv, budget, device="cuda")]

    def step():
        for x, y in zip(dev, (k, v, acc)):
            x.copy_(y)
        return ops.cache_evict(*dev, lens, budget, sinks=4, recent=50, out=None if in_place else (*out, None), handle=h)

    step()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        n = step()
    for i, now in enumerate([[M, 9000], [3, 19001], [701, 0]]):
        acc.copy_(torch.rand(B, nkv, M, generator=torch.Generator().manual_seed(i)))
        lens.copy_(i32(now))
        for x in out if not in_place else []:
            x.zero_()
        g.replay()
        torch.cuda.synchronize()
        host = [x.cpu().clone() for x in (k, v, acc)]
        to = host if in_place else [torch.zeros(x.shape, dtype=x.dtype) for x in out]
        assert n.tolist() == R.evict(*host, None, now, budget, 4, 50, [*to, None])
        for x, y in zip(out, to):
            assert torch.equal(x.cpu(), y), f"replay {i}"
    h.sync()


def test_a_workspace_grows_beside_a_capture():
    """An eager call on another stream allocates its handle's workspace while torch captures: the capture goes on."""
    from flashmlx_b200 import _lib, ops
    lens = [300, 20, 150]
    q, (ck, cv), n = rnd(290, 3, 1, 8, 64), caches(291, 3, 2, 300, 64, lens), i32(lens)
    want = ops.attention_prefix(q, None, None, ck, cv, n)
    side, g, out, x = torch.cuda.Stream(), torch.cuda.CUDAGraph(), torch.zeros_like(q), torch.zeros(4, device="cuda")
    h, cfg = ops.Handle(), _lib.CacheAttnConfig(8, 2, 64, 300, 0, 0, 0.0)
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        x.add_(1.0)
        with torch.cuda.stream(side):
            h.bind_current()
            st = h.lib.fm_attention_prefix(h.h, _lib.C.byref(cfg), q.data_ptr(), None, None, 0, ck.data_ptr(), cv.data_ptr(),
                                           n.data_ptr(), 3, 1, out.data_ptr())
        x.add_(1.0)
    h.check(st)
    h.sync()
    assert torch.equal(out, want)
    g.replay()
    assert x.tolist() == [2.0] * 4


def test_scales_whose_scores_have_no_number_are_refused():
    """The scale times log2(e) has to be a number: beyond, a score of 0 would be 0 times infinity."""
    from flashmlx_b200 import _lib, ops
    q, (ck, cv), n = torch.zeros(2, 1, 4, 64, dtype=BF, device="cuda"), caches(292, 2, 2, 16, 64, [9, 16]), i32([9, 16])
    for scale in (3.0e38, -2.4e38):
        refused(lambda: ops.attention_prefix(q, None, None, ck, cv, n, scale=scale), _lib.FM_EINVAL)
    out = ops.attention_prefix(q, None, None, ck, cv, n, scale=2.3e38)  # scores of 0: the mean of the values
    want, tol, _, _ = R.attention(q, ck, cv, [9, 16])
    held(out, want, tol)


def test_branches_of_a_capture_that_share_a_handle_take_turns():
    """Two streams forked inside a capture, calls on both without a handle given: a replay runs them one after the
    other."""
    from flashmlx_b200 import ops
    lens = [3000, 500, 2100, 77]
    n, data = i32(lens), []
    for i in range(2):
        q, acc = rnd(300 + i, 4, 6, 8, 128), torch.rand(4, 2, 3000, generator=torch.Generator().manual_seed(i)).cuda()
        data.append((q, *caches(302 + 2 * i, 4, 2, 3000, 128, lens), acc))

    def work(q, ck, cv, acc):
        ck, cv, acc = ck.clone(), cv.clone(), acc.clone()
        out = ops.attention_scored(q, ck, cv, n, acc)
        weights = acc.clone()
        return [out, weights, ops.cache_evict(ck, cv, acc, n, 1500, sinks=4, recent=64), ck, cv, acc]

    want = [work(*d) for d in data]
    ops.synchronize()
    g, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(g):
        here = torch.cuda.current_stream()
        side.wait_stream(here)
        got = []
        for _ in range(2):
            got.append((0, work(*data[0])))
            with torch.cuda.stream(side):
                got.append((1, work(*data[1])))
        here.wait_stream(side)
    for _ in range(3):
        for _, outs in got:
            for t in outs:
                t.zero_()
        g.replay()
        torch.cuda.synchronize()
        for i, outs in got:
            for x, y in zip(outs, want[i]):
                assert torch.equal(x.nan_to_num(nan=-7.0), y.nan_to_num(nan=-7.0))
    ops.synchronize()
