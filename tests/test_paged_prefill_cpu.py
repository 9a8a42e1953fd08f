"""CPU checks of the rotary, paged-append and paged-prefill operators: the C entry points refuse what
they cannot take before any CUDA call, the host table of angles, and the division of the attention's
work over CTAs (the arithmetic of csrc/paged_prefill.cuh, restated)."""
import math
import random

import pytest
import torch

from kernelverse_b200 import _lib, ops

P = 1 << 20          # stands for an aligned pointer that is never followed


def _norm_rope(**kw):
    a = dict(q=P, k=P, dtype=_lib.BF16, strides=(512, 128, 128, 128), positions=P, pdt=_lib.I64, cos_sin=P, maxp=16, r=128,
             inter=0, qw=None, kw=None, eps=1e-6, t=2, hq=4, hkv=1, d=128, qo=P, ko=P)
    a.update(kw)
    return _lib.lib().kvb_qk_norm_rope(a["q"], a["k"], a["dtype"], *a["strides"], a["positions"], a["pdt"], a["cos_sin"],
                                       a["maxp"], a["r"], a["inter"], a["qw"], a["kw"], a["eps"], a["t"], a["hq"], a["hkv"],
                                       a["d"], a["qo"], a["ko"], None)


def _append(**kw):
    a = dict(q=P, k=P, v=P, dtype=_lib.BF16, strides=(768, 128) * 3, positions=P, pdt=_lib.I64, slots=P, sdt=_lib.I64,
             cos_sin=P, maxp=16, r=128, inter=0, qw=None, kw=None, eps=1e-6, t=2, hq=4, hkv=1, d=128, kc=P, vc=P,
             cdt=_lib.E4M3, bs=16, nb=4, kbs=2048, vbs=2048, ks=P, vs=P, qo=P)
    a.update(kw)
    return _lib.lib().kvb_rope_paged_kv_append(
        a["q"], a["k"], a["v"], a["dtype"], *a["strides"], a["positions"], a["pdt"], a["slots"], a["sdt"], a["cos_sin"],
        a["maxp"], a["r"], a["inter"], a["qw"], a["kw"], a["eps"], a["t"], a["hq"], a["hkv"], a["d"], a["kc"], a["vc"],
        a["cdt"], a["bs"], a["nb"], a["kbs"], a["vbs"], a["ks"], a["vs"], a["qo"], None)


def _attend(**kw):
    a = dict(q=P, qdt=_lib.BF16, qts=512, kc=P, vc=P, cdt=_lib.BF16, kbs=2048, vbs=2048, ks=None, vs=None, qo=P, sl=P,
             sdt=_lib.I32, bt=P, bts=8, b=1, tq=4, hq=4, hkv=1, d=128, bs=16, nb=4, maxl=128, scale=0.1, out=P, lse=None,
             variant=0, ws=P, wsb=1 << 30)
    a.update(kw)
    return _lib.lib().kvb_paged_prefill_attention_variant(
        a["q"], a["qdt"], a["qts"], a["kc"], a["vc"], a["cdt"], a["kbs"], a["vbs"], a["ks"], a["vs"], a["qo"], a["sl"],
        a["sdt"], a["bt"], a["bts"], a["b"], a["tq"], a["hq"], a["hkv"], a["d"], a["bs"], a["nb"], a["maxl"], a["scale"],
        a["out"], a["lse"], a["variant"], a["ws"], a["wsb"], None)


ARG, SHAPE, ALIGN, DTYPE, WORKSPACE = 1, 2, 3, 4, 7


@pytest.mark.parametrize("bad,code", [
    (dict(q=None), ARG), (dict(cos_sin=None), ARG), (dict(qo=None), ARG), (dict(t=-1), ARG), (dict(hkv=0), ARG),
    (dict(pdt=_lib.F32), DTYPE), (dict(dtype=_lib.I8), DTYPE), (dict(r=130), SHAPE), (dict(r=63), SHAPE),
    (dict(d=127, r=64), SHAPE), (dict(d=2048), SHAPE), (dict(cos_sin=P + 4), ALIGN)])
def test_norm_rope_refusals(bad, code):
    assert _norm_rope(**bad) == code, _lib.lib().kvb_last_error()
    assert b"qk_norm_rope" in _lib.lib().kvb_last_error()


@pytest.mark.parametrize("bad,code", [
    (dict(v=None), ARG), (dict(slots=None), ARG), (dict(ks=None), ARG), (dict(kc=None), ARG), (dict(bs=0), ARG),
    (dict(nb=-1), ARG), (dict(sdt=_lib.BF16), DTYPE), (dict(cdt=_lib.F16), DTYPE), (dict(kbs=2040), SHAPE),
    (dict(r=129), SHAPE)])
def test_append_refusals(bad, code):
    assert _append(**bad) == code, _lib.lib().kvb_last_error()
    assert b"rope_paged_kv_append" in _lib.lib().kvb_last_error()


@pytest.mark.parametrize("bad,code", [
    (dict(q=None), ARG), (dict(bt=None), ARG), (dict(cdt=_lib.E4M3), ARG), (dict(b=-1), ARG), (dict(scale=math.nan), ARG),
    (dict(scale=math.inf), ARG), (dict(variant=3), ARG), (dict(hq=4, hkv=3), SHAPE), (dict(d=136), SHAPE),
    (dict(d=100), SHAPE), (dict(maxl=129), SHAPE), (dict(kbs=1024), SHAPE), (dict(bts=1 << 30, maxl=1 << 28), SHAPE),
    (dict(qdt=_lib.I8), DTYPE), (dict(cdt=_lib.F16), DTYPE), (dict(sdt=_lib.F32), DTYPE), (dict(q=P + 8), ALIGN),
    (dict(qts=516), ALIGN), (dict(kc=P + 8), ALIGN), (dict(out=P + 4), ALIGN), (dict(ws=None), WORKSPACE),
    (dict(wsb=1024), WORKSPACE), (dict(ws=P + 64), WORKSPACE)])
def test_attention_refusals(bad, code):
    assert _attend(**bad) == code, _lib.lib().kvb_last_error()
    assert b"paged_prefill_attention" in _lib.lib().kvb_last_error()


def test_empty_calls_need_no_pointers():
    assert _norm_rope(t=0, q=None, k=None, positions=None, qo=None, ko=None) == 0
    assert _append(t=0, q=None, k=None, v=None, slots=None, positions=None, qo=None) == 0
    assert _attend(b=0, qo=None, sl=None, bt=None) == 0
    assert _attend(tq=0, q=None, out=None) == 0


def test_ops_reject_cpu_tensors():
    x = torch.zeros(2, 4, 64)
    pos = torch.zeros(2, dtype=torch.int64)
    with pytest.raises(ValueError, match="CUDA tensors only"):
        ops.qk_norm_rope(x, x, pos, torch.zeros(8, 64))
    with pytest.raises(ValueError, match="CUDA tensors only"):
        ops.rope_paged_kv_append(x, x, x, torch.zeros(2, 16, 4, 64), torch.zeros(2, 16, 4, 64), pos, pos, torch.zeros(8, 64))
    with pytest.raises(ValueError, match="CUDA tensors only"):
        ops.paged_prefill_attention(x, torch.zeros(2, 16, 4, 64), torch.zeros(2, 16, 4, 64), pos.int(), pos[:1].int(),
                                    pos.int().view(1, 2))


def test_cos_sin_table():
    t = ops.rope_cos_sin(300, 10, base=500.0)
    assert t.dtype == torch.float32 and t.shape == (300, 10)
    for p in (0, 1, 299):
        for n in range(5):
            angle = p * 500.0 ** (-2 * n / 10)
            assert abs(t[p, n].item() - math.cos(angle)) <= 2 ** -24
            assert abs(t[p, 5 + n].item() - math.sin(angle)) <= 2 ** -24
    assert ops.rope_cos_sin(4, 0).shape == (4, 0)
    with pytest.raises(ValueError):
        ops.rope_cos_sin(4, 7)


# ------------------------------------------------------------------------------------------ the division of the work
def floor_sum(n, m, s, b):
    ans = 0
    while n > 0:
        ans += (n - 1) * n // 2 * (s // m) + n * (b // m)
        s, b = s % m, b % m
        y = s * n + b
        if y < m:
            break
        n, b, m, s = y // m, y % m, s, m
    return ans


class Tiles:
    def __init__(self, rt, bku, group):
        self.rt, self.bku, self.group = rt, bku, group

    def count(self, ql):
        return -(-ql * self.group // self.rt)

    def units(self, ql, kl, t):
        last = min((t + 1) * self.rt, ql * self.group) - 1
        x = (kl - ql) * self.group + last
        return 1 if x < 0 else x // (self.group * self.bku) + 1

    def before(self, ql, kl, t):
        if t == 0:
            return 0
        n, total, full = self.count(ql), 0, t
        if t == n:
            total, full = self.units(ql, kl, n - 1), full - 1
        if full == 0:
            return total
        total += full
        x0 = (kl - ql) * self.group + self.rt - 1
        skip = 0 if x0 >= 0 else min(full, (-x0 + self.rt - 1) // self.rt)
        if full > skip:
            total += floor_sum(full - skip, self.group * self.bku, self.rt, x0 + skip * self.rt)
        return total


@pytest.mark.parametrize("seed", range(40))
def test_units_before_a_tile_is_their_sum(seed):
    rng = random.Random(seed)
    tiles = Tiles(rng.choice((64, 128, 256)), rng.choice((32, 64, 128, 256)), rng.choice((1, 2, 3, 4, 5, 7, 8, 16, 71)))
    ql = rng.choice((1, 2, 5, 64, 100, rng.randrange(1, 1500)))
    kl = rng.choice((0, 1, ql, max(0, ql - rng.randrange(1, 300)), ql + rng.randrange(0, 5000)))
    total = 0
    for t in range(tiles.count(ql)):
        assert tiles.before(ql, kl, t) == total
        # the tile's last row sees keys 0 .. kl - ql + its token, all inside its units, and no unit is idle
        last_token = (min((t + 1) * tiles.rt, ql * tiles.group) - 1) // tiles.group
        keys = max(0, kl - ql + last_token + 1)
        assert tiles.units(ql, kl, t) == max(1, -(-keys // tiles.bku))
        total += tiles.units(ql, kl, t)
    assert tiles.before(ql, kl, tiles.count(ql)) == total


@pytest.mark.parametrize("seed", range(20))
def test_shares_cover_every_unit_once_and_parts_are_consecutive(seed):
    """CTA c of n takes units [c W / n, (c + 1) W / n): every CTA has at least one, an item that is cut is begun by
    one CTA and continued by the ones right after it, and each continues at most one item, begins at most one cut item."""
    rng = random.Random(100 + seed)
    items = [rng.randrange(1, rng.choice((2, 8, 300))) for _ in range(rng.randrange(1, 60))]
    total, grid = sum(items), rng.choice((1, 7, 148, 296))
    ctas = min(total, grid)
    bound = [total * c // ctas for c in range(ctas + 1)]
    assert bound[0] == 0 and bound[-1] == total and all(a < b for a, b in zip(bound, bound[1:]))
    start, continued, begun = 0, set(), set()
    for n in items:
        owners = [c for c in range(ctas) if bound[c] < start + n and bound[c + 1] > start]
        assert owners == list(range(owners[0], owners[-1] + 1))
        last = ((start + n) * ctas - 1) // total                     # pg_cta_of(start + n - 1)
        while last + 1 < ctas and total * (last + 1) // ctas <= start + n - 1:
            last += 1
        while last > 0 and total * last // ctas > start + n - 1:
            last -= 1
        assert last == owners[-1]
        if len(owners) > 1:
            assert owners[0] not in begun and not continued & set(owners[1:])
            begun.add(owners[0])
            continued |= set(owners[1:])
        start += n
