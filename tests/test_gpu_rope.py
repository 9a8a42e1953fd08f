"""GPU tests of qk_norm_rope and rope_paged_kv_append against the float64 oracle.

Tolerances.  A value is computed in float32 and rounded once: half a step of its type, plus the
float32 errors relative to |y_i c| + |y_j s| (the oracle's `size`).  Those are at most: the mean of up
to 1024 squares, each addition 2^-24 relative, pairwise in part (<= 40 additions in a row here), halved by
the square root; rsqrt (2^-22); three products and one sum (2^-24 each): below 32 * 2^-24 = 2^-19.  An
e4m3 code is the rounding of a quotient with that error: its value is within half a step (2^-4
relative, 2^-10 absolute below the normal range) and 2^-19 of the scaled size, times the scale.
"""
import numpy as np
import pytest
import torch

from gpu_util import dev, host, require_gpu, seeded
from oracle import numerics, rope

pytestmark = pytest.mark.gpu

DT = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-6


@pytest.fixture(autouse=True)
def _gpu():
    require_gpu()


def _ops():
    from kernelverse_b200 import ops
    return ops


def _case(seed, t, hq, hkv, d, r, dt, maxp=500, fused=True):
    rng = seeded(seed)
    x = dev(rng.standard_normal((t, (hq + 2 * hkv) * d)).astype(np.float32), DT[dt])
    q = x[:, :hq * d].view(t, hq, d)
    k = x[:, hq * d:(hq + hkv) * d].view(t, hkv, d)
    v = x[:, (hq + hkv) * d:].view(t, hkv, d)
    if not fused:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    pos = dev(rng.integers(0, maxp, t).astype(np.int64))
    return q, k, v, pos, _ops().rope_cos_sin(maxp, r, device="cuda")


def _weights(seed, d, dt):
    rng = seeded(seed + 999)
    return tuple(dev((1 + 0.2 * rng.standard_normal(d)).astype(np.float32), DT[dt]) for _ in range(2))


def _near(got, ref, size, dtype):
    half = torch.finfo(dtype).eps / 2
    tiny = {torch.float16: 2.0 ** -25, torch.bfloat16: 0.0, torch.float32: 0.0}[dtype]     # below fp16's normal range
    err = np.abs(host(got).astype(np.float64) - ref)
    bound = half * np.abs(ref) + (1 + half) * 2.0 ** -19 * size + tiny
    assert (err <= bound).all(), f"{(err / np.maximum(bound, 1e-300)).max()} times the bound"


def _check(seed, t, hq, hkv, d, r, dt, interleaved, norm, fused=True):
    q, k, _, pos, table = _case(seed, t, hq, hkv, d, r, dt, fused=fused)
    qw, kw = _weights(seed, d, dt) if norm else (None, None)
    qo, ko = _ops().qk_norm_rope(q, k, pos, table, qw, kw, EPS, interleaved)
    assert qo.is_contiguous() and ko.is_contiguous() and qo.dtype == ko.dtype == DT[dt]
    assert qo.shape == (t, hq, d) and ko.shape == (t, hkv, d)
    for got, x, w in ((qo, q, qw), (ko, k, kw)):
        ref, size = rope.norm_rope(host(x), None if w is None else host(w), host(pos), host(table), EPS, interleaved)
        _near(got, ref, size, DT[dt])


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("d,r", [(128, 128), (64, 32), (80, 80), (80, 40), (256, 64), (96, 0), (40, 20), (6, 4), (130, 130)])
def test_norm_rope(dt, interleaved, norm, d, r):
    """Vector widths 8 and 4 and the element-wise kernel, whole, partial and no rotation, lanes left over."""
    _check(d * 7 + r, 13, 5, 2, d, r, dt, interleaved, norm)


@pytest.mark.parametrize("t,hq,hkv", [(1, 1, 1), (1, 32, 8), (2, 7, 1), (300, 9, 3), (2500, 32, 8)])
@pytest.mark.parametrize("fused", [True, False])
def test_norm_rope_sizes(t, hq, hkv, fused):
    """One token up to enough for four heads a team; heads that are not a multiple of four."""
    _check(t + hq, t, hq, hkv, 64, 64, "bf16", False, True, fused)


def test_norm_rope_strides_and_alignment():
    """Heads apart by more than they are long, and rows off the 16-byte grid (the element-wise kernel): the
    same numbers as on packed copies."""
    ops, rng = _ops(), seeded(5)
    table = ops.rope_cos_sin(64, 64, device="cuda")
    pos = dev(rng.integers(0, 64, 9).astype(np.int32))
    for wide, at in ((72, 0), (72, 8), (71, 3), (65, 1)):
        x = dev(rng.standard_normal((9, 6, wide)).astype(np.float32), torch.bfloat16)
        q, k = x[:, :4, at:at + 64] if wide > 64 + at else x[:, :4, :64], x[:, 4:, :64]
        got = ops.qk_norm_rope(q, k, pos, table)
        want = ops.qk_norm_rope(q.contiguous(), k.contiguous(), pos, table)
        for g, w, src in zip(got, want, (q, k)):
            ref, size = rope.norm_rope(host(src), None, host(pos), host(table), EPS, False)
            _near(g, ref, size, torch.bfloat16)
            _near(w, ref, size, torch.bfloat16)


def test_norm_rope_large_and_tiny_heads():
    """Heads of zeros (eps alone under the root), of 2^-60 and of 2^60."""
    ops = _ops()
    x = torch.randn((3, 4, 64), device="cuda")
    x[0] = 0
    x[1] *= 2.0 ** -60
    x[2] *= 2.0 ** 60
    w = torch.ones(64, device="cuda")
    pos = torch.arange(3, device="cuda")
    table = ops.rope_cos_sin(8, 64, device="cuda")
    got, _ = ops.qk_norm_rope(x, x, pos, table, w, w, EPS)
    ref, size = rope.norm_rope(host(x), host(w), host(pos), host(table), EPS, False)
    _near(got, ref, size, torch.float32)


def _cache(seed, nb, bs, hkv, d, cache, scale, joint):
    """K and V caches with known contents; ``joint``: views of one [nb, 2, bs, hkv, d] tensor."""
    rng = seeded(seed + 31)
    if cache == "e4m3":
        raw = dev(rng.integers(0, 255, (nb, 2, bs, hkv, d)).astype(np.uint8)).view(torch.float8_e4m3fn)
    else:
        raw = dev(rng.standard_normal((nb, 2, bs, hkv, d)).astype(np.float32), DT[cache])
    if joint:
        return raw[:, 0], raw[:, 1]
    return raw.view(torch.uint8)[:, 0].contiguous().view(raw.dtype), raw.view(torch.uint8)[:, 1].contiguous().view(raw.dtype)


def _bytes(t):
    return t.contiguous().view(torch.uint8).cpu().numpy()


def _append(seed, t, hq, hkv, d, r, bs, dt, cache, interleaved, norm, joint=False, idx=np.int64, padded=0):
    q, k, v, pos, table = _case(seed, t, hq, hkv, d, r, dt)
    qw, kw = _weights(seed, d, dt) if norm else (None, None)
    rng = seeded(seed + 77)
    nb = t // bs + 3
    ks = vs = None
    if cache == "e4m3":
        ks, vs = (dev((rng.random(hkv) * 0.01 + 0.005).astype(np.float32)) for _ in range(2))
    kc, vc = _cache(seed, nb, bs, hkv, d, cache, ks, joint)
    slots = rng.permutation(nb * bs)[:t].astype(idx)
    if padded:
        slots[rng.permutation(t)[:padded]] = -1
    before = _bytes(kc), _bytes(vc)
    qo = _ops().rope_paged_kv_append(q, k, v, kc, vc, dev(slots), pos, table, ks, vs, qw, kw, EPS, interleaved)
    ref, size = rope.norm_rope(host(q), None if qw is None else host(qw), host(pos), host(table), EPS, interleaved)
    _near(qo, ref, size, DT[dt])
    kref, ksize = rope.norm_rope(host(k), None if kw is None else host(kw), host(pos), host(table), EPS, interleaved)
    live = slots >= 0
    blk, row = slots[live] // bs, slots[live] % bs
    for c, was, x, sz, s in ((kc, before[0], kref, ksize, ks), (vc, before[1], host(v).astype(np.float64), None, vs)):
        now = _bytes(c)
        untouched = np.ones((nb, bs), bool)
        untouched[blk, row] = False
        np.testing.assert_array_equal(now[untouched], was[untouched])       # every other slot keeps its bytes
        if cache != "e4m3":
            got = c[torch.from_numpy(blk).cuda().long(), torch.from_numpy(row).cuda().long()]
            if sz is None:
                np.testing.assert_array_equal(host(got), x[live])           # values are copied
            else:
                _near(got, x[live], sz[live], DT[dt])
            continue
        got = numerics.e4m3_decode(now[blk, row]).astype(np.float64)
        sc = host(s).astype(np.float64)[None, :, None]
        want = np.clip(x[live] / sc, -448, 448)
        if sz is None:                                                       # the correctly rounded quotient's code
            exact = numerics.e4m3_quantize(x[live].astype(np.float32), host(s)[None, :, None])
            np.testing.assert_array_equal(now[blk, row] & 0x7f, exact & 0x7f)
            np.testing.assert_array_equal(got, numerics.e4m3_decode(exact).astype(np.float64))
        else:
            bound = np.maximum(2.0 ** -4 * np.abs(want), 2.0 ** -10) + (1 + 2.0 ** -4) * 2.0 ** -19 * sz[live] / sc
            assert (np.abs(got - want) <= bound).all()


@pytest.mark.parametrize("dt,cache", [("bf16", "bf16"), ("bf16", "e4m3"), ("fp16", "fp16"), ("fp16", "e4m3"), ("fp32", "fp32"),
                                      ("fp32", "e4m3")])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,r,bs", [(128, 128, 16), (64, 32, 20), (80, 40, 1), (6, 4, 7), (36, 36, 12)])
def test_append(dt, cache, interleaved, d, r, bs):
    _append(d + bs, 29, 6, 2, d, r, bs, dt, cache, interleaved, interleaved, padded=4)


@pytest.mark.parametrize("joint", [False, True])
@pytest.mark.parametrize("cache", ["bf16", "e4m3"])
def test_append_joint_cache_and_int32_slots(cache, joint):
    """Keys and values of a block side by side in one tensor: the caches are views with wide block strides."""
    _append(3, 50, 8, 2, 128, 128, 16, "bf16", cache, False, True, joint=joint, idx=np.int32)


@pytest.mark.parametrize("t", [1, 3000])
def test_append_one_token_and_many(t):
    _append(8, t, 32, 8, 128, 128, 16, "bf16", "e4m3", False, False)


def test_append_slot_offsets_past_32_bits():
    """A cache of more than 2^31 elements: the far slots are written where they belong."""
    ops = _ops()
    nb, bs, h, d = 17000, 16, 64, 128                     # 2.2e9 codes a cache
    kc = torch.zeros((nb, bs, h, d), dtype=torch.uint8, device="cuda")
    q, k, v, pos, table = _case(4, 3, 64, 64, 128, 128, "bf16")
    one = torch.ones(h, device="cuda")
    slots = torch.tensor([nb * bs - 1, 0, 1 << 18], device="cuda")
    ops.rope_paged_kv_append(q, k, v, kc, kc.clone(), slots, pos, table, one, one)
    ref, size = rope.norm_rope(host(k), None, host(pos), host(table), EPS, False)
    got = numerics.e4m3_decode(kc.view(nb * bs, h, d)[slots].cpu().numpy()).astype(np.float64)
    assert (np.abs(got - ref) <= np.maximum(2.0 ** -4 * np.abs(ref), 2.0 ** -10) + 2.0 ** -18 * size).all()
    assert int((kc.view(nb * bs, -1).any(1)).sum()) == 3


def test_bad_positions_and_slots_are_flagged():
    """NaN heads and an untouched cache for a position outside the table; a slot past the cache is skipped;
    both set bit 1, and the other tokens come out as ever."""
    from kernelverse_b200 import _lib
    ops = _ops()
    q, k, v, pos, table = _case(6, 5, 4, 2, 64, 64, "bf16", maxp=100)
    want, wantk = ops.qk_norm_rope(q, k, pos, table)
    assert _lib.lib().kvb_device_status(1) == 0
    bad = pos.clone()
    bad[1], bad[3] = -1, 100
    got, gotk = ops.qk_norm_rope(q, k, bad, table)
    assert _lib.lib().kvb_device_status(1) == 2
    good = torch.tensor([0, 2, 4], device="cuda")
    assert torch.equal(got[good], want[good]) and torch.equal(gotk[good], wantk[good])
    assert got[[1, 3]].isnan().all() and gotk[[1, 3]].isnan().all()
    kc = torch.zeros((2, 4, 2, 64), dtype=torch.bfloat16, device="cuda")
    vc = torch.zeros_like(kc)
    slots = torch.tensor([0, 1, 8, 3, 1 << 40], device="cuda")
    qo = ops.rope_paged_kv_append(q, k, v, kc, vc, slots, bad, table)
    assert _lib.lib().kvb_device_status(1) == 2
    assert torch.equal(qo[good], want[good]) and qo[[1, 3]].isnan().all()
    assert torch.equal(kc.view(8, 2, 64)[0], wantk[0]) and not kc.view(8, 2, 64)[1:].any()
    assert torch.equal(vc.view(8, 2, 64)[0], v[0]) and not vc.view(8, 2, 64)[1:].any()


def test_no_tokens():
    ops = _ops()
    e = torch.empty((0, 4, 64), dtype=torch.bfloat16, device="cuda")
    kc = torch.zeros((2, 4, 4, 64), dtype=torch.bfloat16, device="cuda")
    i = torch.empty(0, dtype=torch.int64, device="cuda")
    table = ops.rope_cos_sin(4, 64, device="cuda")
    assert ops.qk_norm_rope(e, e, i, table)[0].shape == (0, 4, 64)
    assert ops.rope_paged_kv_append(e, e, e, kc, kc.clone(), i, i, table).shape == (0, 4, 64) and not kc.any()


def test_refusals():
    ops = _ops()
    q, k, v, pos, table = _case(1, 4, 4, 2, 64, 64, "bf16")
    kc = torch.zeros((2, 4, 2, 64), dtype=torch.bfloat16, device="cuda")
    slots = torch.arange(4, device="cuda")
    with pytest.raises(TypeError, match="share a dtype"):
        ops.qk_norm_rope(q, k.float(), pos, table)
    with pytest.raises(ValueError, match="positions"):
        ops.qk_norm_rope(q, k, pos[:3], table)
    with pytest.raises(TypeError, match="cos_sin"):
        ops.qk_norm_rope(q, k, pos, table.double())
    with pytest.raises(ValueError, match="norm weights"):
        ops.qk_norm_rope(q, k, pos, table, torch.ones(64, device="cuda"))
    with pytest.raises(TypeError, match="int32 or int64"):
        ops.qk_norm_rope(q, k, pos.float(), table)
    with pytest.raises(RuntimeError, match="rotary_dim"):
        ops.qk_norm_rope(q, k, pos, ops.rope_cos_sin(500, 66, device="cuda"))
    with pytest.raises(ValueError, match="scales"):
        ops.rope_paged_kv_append(q, k, v, kc, kc.clone(), slots, pos, table, torch.ones(2, device="cuda"), None)
    with pytest.raises(ValueError, match="k_scale and v_scale"):
        c = kc.to(torch.float8_e4m3fn)
        ops.rope_paged_kv_append(q, k, v, c, c.clone(), slots, pos, table)
    with pytest.raises(TypeError, match="e4m3"):
        ops.rope_paged_kv_append(q, k, v, kc.half(), kc.half(), slots, pos, table)
    with pytest.raises(ValueError, match="blocks of k_cache"):
        ops.rope_paged_kv_append(q, k, v, kc.transpose(1, 2).contiguous().transpose(1, 2), kc, slots, pos, table)
    with pytest.raises(ValueError, match="slot_mapping"):
        ops.rope_paged_kv_append(q, k, v, kc, kc.clone(), slots[:2], pos, table)


def test_captured_and_replayed_on_another_stream():
    """A captured append replays on changed inputs, and gives what an eager call gives."""
    ops = _ops()
    q, k, v, pos, table = _case(9, 40, 8, 2, 128, 128, "bf16")
    ks = torch.full((2,), 0.02, device="cuda")
    kc = torch.zeros((4, 16, 2, 128), dtype=torch.uint8, device="cuda")
    vc, kc2, vc2 = kc.clone(), kc.clone(), kc.clone()
    slots = torch.randperm(64, device="cuda")[:40]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        ops.rope_paged_kv_append(q, k, v, kc, vc, slots, pos, table, ks, ks)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            qo = ops.rope_paged_kv_append(q, k, v, kc, vc, slots, pos, table, ks, ks)
        pos.copy_((pos + 17) % 500)
        kc.zero_(), vc.zero_()
        g.replay()
        want = ops.rope_paged_kv_append(q, k, v, kc2, vc2, slots, pos, table, ks, ks)
    s.synchronize()
    assert torch.equal(qo, want) and torch.equal(kc, kc2) and torch.equal(vc, vc2)


def _special(x):
    """Infinities, NaN and signed zeros strewn over the elements."""
    n = torch.arange(x.numel(), device=x.device).view(x.shape)
    for k, value in enumerate((float("inf"), float("-inf"), float("nan"), -0.0, 0.0)):
        x = torch.where(n % 11 == 2 * k, torch.full_like(x, value), x)
    return x


def _same(a, b):
    """Equal values and signs of zeros; NaN equals NaN."""
    a, b = a.float(), b.float()
    return bool((((a == b) & (a.signbit() == b.signbit())) | (a.isnan() & b.isnan())).all())


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("t", [5, 3000])
@pytest.mark.parametrize("d,r", [(64, 0), (64, 32), (80, 40), (96, 16), (40, 24), (128, 8), (6, 4)])
def test_elements_past_the_rotary_dim_pass_whatever_they_are(dt, interleaved, t, d, r):
    """Infinities, NaN and -0.0 behind the rotary dim come out as they are, and change nothing else: in the vector
    kernels (one and two heads a team), in the element-wise one (rows off the 16-byte grid), and through the append."""
    ops, rng = _ops(), seeded(d + r)
    hq, hkv = 5, 3
    table = ops.rope_cos_sin(64, r, device="cuda")
    pos = dev(rng.integers(0, 64, t).astype(np.int64))
    slots = torch.randperm(t, device="cuda")
    for wide in (d, d + 1):
        x = torch.zeros((t, hq + 2 * hkv, wide), dtype=DT[dt], device="cuda")[..., :d]
        x.copy_(torch.from_numpy(rng.standard_normal((t, hq + 2 * hkv, d)).astype(np.float32)))
        plain = x[:, :hq].clone(), x[:, hq:hq + hkv].clone()
        x[..., r:] = _special(x[..., r:])
        q, k, v = x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]
        kc = torch.zeros((t, 1, hkv, d), dtype=DT[dt], device="cuda")
        vc = kc.clone()
        got = *ops.qk_norm_rope(q, k, pos, table, interleaved=interleaved), \
            ops.rope_paged_kv_append(q, k, v, kc, vc, slots, pos, table, interleaved=interleaved), kc[slots, 0]
        for out, src, fin in zip(got, (q, k, q, k), plain + plain):
            assert _same(out[..., r:], src[..., r:])
            ref, size = rope.norm_rope(host(fin), None, host(pos), host(table), EPS, interleaved)
            _near(out[..., :r], ref[..., :r], size[..., :r], DT[dt])
        assert _same(vc[slots, 0], v)


@pytest.mark.parametrize("interleaved", [False, True])
def test_zeros_keep_their_signs_behind_the_rotary_dim_of_normalised_heads(interleaved):
    ops = _ops()
    x = torch.randn((4, 6, 64), device="cuda")
    x[..., 33::5] = -0.0
    x[..., 34::5] = 0.0
    w = torch.ones(64, device="cuda")
    out, _ = ops.qk_norm_rope(x, x, torch.arange(4, device="cuda"), ops.rope_cos_sin(8, 32, device="cuda"), w, w, EPS, interleaved)
    zero = x[..., 32:] == 0
    assert _same(out[..., 32:][zero], x[..., 32:][zero])


def _codes(x, scale):
    """The value of e4m3(clamp(x / scale, +-448)) in float32; NaN for NaN."""
    with np.errstate(all="ignore"):
        q = np.clip(x.astype(np.float32) / scale.astype(np.float32)[None, :, None], np.float32(-448), np.float32(448))
    out = numerics.e4m3_decode(numerics.e4m3_encode(np.nan_to_num(q, nan=0.0)))
    return np.where(np.isnan(q), np.float32(np.nan), out)


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("t", [6, 4000])
@pytest.mark.parametrize("d,wide", [(64, 64), (20, 20), (64, 65)])
def test_append_saturates_what_is_out_of_range(dt, t, d, wide):
    """Infinities and quotients past float32 become +-448 and NaN stays NaN, for scales of a cache's size and for the
    smallest and largest: vectors of eight and of four, one and two heads a team, and the element-wise kernel."""
    ops, rng = _ops(), seeded(d + t)
    scale = np.array([0.005, 1.0, 2.0 ** -125, 1e-38, 2.0 ** -120, 2.0 ** 120, 2.0 ** 125], np.float32)
    hkv = len(scale)
    x = torch.zeros((t, 2 * hkv, wide), dtype=DT[dt], device="cuda")[..., :d]
    x.copy_(torch.from_numpy(rng.standard_normal((t, 2 * hkv, d)).astype(np.float32)))
    top = torch.finfo(DT[dt]).max
    flat = torch.arange(x.numel(), device="cuda").view(x.shape)
    for i, value in enumerate((float("inf"), float("-inf"), float("nan"), top, -top, top / 16, 0.0, -0.0)):
        x[flat % 17 == 2 * i] = value
    k, v = x[:, :hkv], x[:, hkv:]
    kc = torch.zeros((t, 1, hkv, d), dtype=torch.uint8, device="cuda")
    vc = kc.clone()
    slots = torch.randperm(t, device="cuda")
    sc = dev(scale)
    ops.rope_paged_kv_append(k, k, v, kc, vc, slots, torch.zeros(t, dtype=torch.int64, device="cuda"),
                             torch.zeros((1, 0), device="cuda"), sc, sc)
    for cache, src in ((kc, k), (vc, v)):
        got = numerics.e4m3_decode(cache[slots, 0].cpu().numpy())
        np.testing.assert_array_equal(got, _codes(host(src.contiguous()), scale))


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("hq,hkv,d,r", [(5, 3, 64, 64), (4, 1, 80, 40), (7, 2, 20, 16), (6, 3, 128, 64)])
def test_long_inputs_two_heads_a_team(dt, interleaved, hq, hkv, d, r):
    """Long inputs give a team two heads: teams with a query and a key head, a key and a value head, and one head only;
    vectors of eight and of four; partial rotation; positions out of range keep to their own tokens."""
    from kernelverse_b200 import _lib
    t = 10000
    _check(d + hq, t, hq, hkv, d, r, dt, interleaved, True)
    _append(d + hkv, t, hq, hkv, d, r, 16, dt, dt, interleaved, False, padded=900)
    _append(d + hkv, t, hq, hkv, d, r, 16, dt, "e4m3", interleaved, True)
    ops = _ops()
    q, k, _, pos, table = _case(1, t, hq, hkv, d, r, dt)
    qw, kw = _weights(1, d, dt)
    want = ops.qk_norm_rope(q, k, pos, table, qw, kw, EPS, interleaved)
    bad = pos.clone()
    bad[::7], bad[3::70] = 500, -1
    out = (bad < 0) | (bad >= 500)
    assert _lib.lib().kvb_device_status(1) == 0
    got = ops.qk_norm_rope(q, k, bad, table, qw, kw, EPS, interleaved)
    assert _lib.lib().kvb_device_status(1) == 2
    for g, w in zip(got, want):
        assert g[out].isnan().all() and torch.equal(g[~out], w[~out])
