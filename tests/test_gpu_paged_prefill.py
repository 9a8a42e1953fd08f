"""GPU tests of paged_prefill_attention against the float64 oracle, and of the serving sequence that
appends a chunk to the paged cache and attends over it.

Tolerances, with the oracle's `weight` (the row's average of |v|, A below) and `reach` (the largest
|scale| sum |q_d k_d| of the row, Z below):

* products of 16-bit operands are exact in float32 and their sums lose at most 2^-23 relative per
  addition (tensor cores may truncate), D of them: the logits are off by D 2^-23 Z; float32 operands go
  through three TF32 products, which drop terms of 2^-21 Z.  A logit off by e moves the output by 2 e A.
* the exponential is good to 2^-18 (a wide bound: the hardware's is good to 2^-22) and its argument, below 32
  for weights that count, to 2^-24 relative, 2^-19: together under 2^-17 A;
* P is rounded to the operand type of the second product (half a step, relative): eps / 2 A, and float32
  again drops 2^-21 A; weights below that type's normal range (float16: 2^-21 of the largest) lose at most
  2^-32 of the largest each: L 2^-32 max|v|, under 2^-17 for the lengths here (max|v| < 8);
* sums over L keys: L 2^-23 A;
* the result is rounded once: eps / 2 |out|.
The log-sum-exp is off by the logits' error, the exponentials' 2^-17, the sum's L 2^-23 and 2^-22 |lse|
of its own.
"""
import numpy as np
import pytest
import torch

from gpu_util import dev, host, require_gpu, seeded
from oracle import attention, numerics, rope

pytestmark = pytest.mark.gpu

DT = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(autouse=True)
def _gpu():
    require_gpu()


def _ops():
    from kernelverse_b200 import ops
    return ops


class Case:
    """A ragged batch over a paged cache; the cache's unused rows hold NaN."""

    def __init__(self, seed, chunks, contexts, hq, hkv, d, bs, dt, cache=None, spread=1.0, joint=False, tail=0):
        rng = seeded(seed)
        cache = cache or dt
        self.dt, self.cache, self.bs, self.d = dt, cache, bs, d
        self.chunks, self.contexts = list(chunks), list(contexts)
        qo = np.concatenate([[0], np.cumsum(chunks)]).astype(np.int32)
        pages = [-(-c // bs) for c in contexts]
        nb = sum(pages) + 2
        order = rng.permutation(nb).astype(np.int32)
        bt = np.full((len(pages), max(max(pages), 1) + 1), -7, np.int32)      # unused entries point nowhere
        at = 0
        for b, n in enumerate(pages):
            bt[b, :n] = order[at:at + n]
            at += n
        self.q = dev((spread * rng.standard_normal((int(qo[-1]) + tail, hq, d))).astype(np.float32), DT[dt])
        used = np.zeros((nb, bs), bool)
        for b, c in enumerate(contexts):
            for t in range(c):
                used[bt[b, t // bs], t % bs] = True
        kv = rng.standard_normal((nb, 2, bs, hkv, d)).astype(np.float32)
        self.ks = self.vs = None
        if cache == "e4m3":
            sc = (rng.random((2, hkv)) * 0.01 + 0.005).astype(np.float32)
            codes = numerics.e4m3_encode(np.clip(kv / sc[None, :, None, :, None], -448, 448).astype(np.float32))
            codes[~np.broadcast_to(used[:, None], codes.shape[:3])] = 0x7f     # NaN
            raw = dev(codes).view(torch.float8_e4m3fn)
            self.ks, self.vs = dev(sc[0]), dev(sc[1])
            val = numerics.e4m3_decode(codes).astype(np.float64) * sc[None, :, None, :, None].astype(np.float64)
        else:
            raw = dev(kv, DT[cache])
            raw[~torch.from_numpy(np.ascontiguousarray(np.broadcast_to(used[:, None], kv.shape[:3]))).cuda()] = float("nan")
            val = host(raw).astype(np.float64)
        self.k_val, self.v_val = val[:, 0], val[:, 1]
        if joint:
            self.kc, self.vc = raw[:, 0], raw[:, 1]
        else:
            u = raw.view(torch.uint8)
            self.kc, self.vc = (u[:, i].contiguous().view(raw.dtype) for i in (0, 1))
        self.qo_h, self.bt_h = qo, bt
        self.qo, self.bt = dev(qo), dev(bt)
        self.lens = dev(np.array(contexts, np.int32))

    def run(self, **kw):
        return _ops().paged_prefill_attention(self.q, self.kc, self.vc, self.qo, self.lens, self.bt, k_scale=self.ks,
                                              v_scale=self.vs, **kw)

    def check(self, variant, scale=None, **kw):
        scale = self.d ** -0.5 if scale is None else scale
        out, lse = self.run(scale=scale, return_lse=True, _variant=variant, **kw)
        assert out.dtype == DT[self.dt] and out.shape == self.q.shape and lse.shape == self.q.shape[:2]
        n = int(self.qo_h[-1])
        ref, rlse, weight, reach = attention.paged_prefill_attention(host(self.q)[:n], self.k_val, self.v_val, self.qo_h,
                                                                     self.contexts, self.bt_h, scale)
        half = torch.finfo(DT[self.dt]).eps / 2
        f32 = self.dt == "fp32"
        length = max(self.contexts + [1])
        logit = reach * (self.d * 2.0 ** -23 + (2.0 ** -21 if f32 else 0))
        bound = half * np.abs(ref) + (2 * logit[..., None] + (2.0 ** -21 if f32 else half) + 2.0 ** -17 + length * 2.0 ** -23) * weight
        bound = bound + (2.0 ** -17 if self.dt == "fp16" or self.cache == "e4m3" else 0.0) * (weight > 0)
        bound = bound * (1 + half)
        err = np.abs(host(out)[:n].astype(np.float64) - ref)
        assert (err <= bound).all(), f"{np.nanmax(err / np.maximum(bound, 1e-30))} times the bound; nan {np.isnan(err).sum()}"
        got = host(lse)[:n].astype(np.float64)
        empty = np.isinf(rlse)
        assert np.array_equal(np.isneginf(got), empty)
        lb = logit + length * 2.0 ** -23 + 2.0 ** -17 + 2.0 ** -22 * np.abs(np.where(empty, 0, rlse))
        assert (np.abs(np.where(empty, 0, got) - np.where(empty, 0, rlse)) <= lb).all()
        return out


# (query type, cache type, 1 = mma.sync / 2 = tcgen05)
KINDS = [("fp32", "fp32", 1), ("fp32", "e4m3", 1), ("fp16", "fp16", 1), ("bf16", "bf16", 1), ("bf16", "e4m3", 1),
         ("fp16", "e4m3", 1), ("fp16", "fp16", 2), ("bf16", "bf16", 2), ("bf16", "e4m3", 2), ("fp16", "e4m3", 2)]


@pytest.mark.parametrize("dt,cache,variant", KINDS)
@pytest.mark.parametrize("chunks,contexts,hq,hkv,d,bs", [
    ([1, 1, 1], [1, 40, 700], 8, 2, 128, 16),            # one token each: decode
    ([4, 3], [900, 130], 8, 2, 128, 16),                 # drafted tokens
    ([70, 1, 130, 33], [200, 999, 130, 600], 8, 2, 64, 16),      # decodes and prefills at once
    ([40, 9], [100, 9], 6, 2, 128, 20),                  # groups of 3; pages that end inside a tile
    ([50], [333], 7, 1, 80, 12),                         # groups of 7, head_dim 80, pages of 12
    ([129, 64], [129, 64], 4, 4, 96, 8),                 # no shared heads, head_dim 96
    ([30], [300], 16, 1, 64, 1),                         # pages of one token, one KV head
    ([300], [1000], 2, 1, 128, 128),                     # large pages
])
def test_shapes(dt, cache, variant, chunks, contexts, hq, hkv, d, bs):
    if variant == 2 and bs % 4:
        pytest.skip("pages that are not a multiple of four tokens run on the mma.sync kernel")
    Case(hq * 100 + d + bs, chunks, contexts, hq, hkv, d, bs, dt, cache).check(variant)


@pytest.mark.parametrize("dt,cache,variant", [("fp32", "fp32", 1), ("bf16", "bf16", 1), ("bf16", "bf16", 2), ("bf16", "e4m3", 2)])
@pytest.mark.parametrize("chunks,contexts", [
    ([1], [1]), ([5], [0]), ([5], [3]), ([0, 3, 0], [0, 3, 50]), ([0, 7], [20, 7]), ([200, 1], [70, 0]),
    ([63, 64, 65], [63, 64, 65]), ([127, 128, 129], [255, 256, 257]), ([255, 256, 257], [257, 256, 511]),
    ([1, 1], [127, 128]), ([1, 1], [129, 256]), ([2], [513]),
])
def test_edges(dt, cache, variant, chunks, contexts):
    """Empty requests, chunks longer than their context (rows that see nothing), lengths one below, at and
    above the tiles of rows and of keys."""
    Case(sum(chunks) + sum(contexts), chunks, contexts, 4, 2, 64, 16, dt, cache).check(variant)


@pytest.mark.parametrize("dt,variant", [("fp32", 1), ("bf16", 1), ("fp16", 1)])
@pytest.mark.parametrize("d", [8, 24, 32, 40, 72, 104, 112])
def test_head_dims(dt, variant, d):
    Case(d, [20, 1], [90, 70], 4, 2, d, 16, dt).check(variant)


@pytest.mark.parametrize("cache", ["bf16", "e4m3"])
@pytest.mark.parametrize("d", [64, 80, 96, 112, 128])
@pytest.mark.parametrize("bs", [4, 12, 24, 64, 384])
def test_tcgen05_head_dims_and_pages(cache, d, bs):
    """Every head_dim of the tcgen05 kernel with pages of 4 to 384 tokens: boxes of 4 to 128 keys."""
    Case(d + bs, [150, 1, 9], [460, 700, 9], 4, 2, d, bs, "bf16", cache).check(2)


@pytest.mark.parametrize("variant", [1, 2])
@pytest.mark.parametrize("hq,hkv", [(71, 1), (5, 5), (130, 1), (24, 3)])
def test_head_counts(hq, hkv, variant):
    """More heads on one KV head than a tile has rows, and groups that no tile is a multiple of."""
    Case(hq, [7, 1], [60, 90], hq, hkv, 64, 16, "bf16").check(variant)


@pytest.mark.parametrize("variant", [1, 2])
@pytest.mark.parametrize("scale", [0.0, -0.2, 3.0])
def test_scales_and_peaked_rows(scale, variant):
    """Equal weights, a negative scale, and logits far apart (one key takes all)."""
    Case(5, [33, 1], [150, 200], 4, 2, 64, 16, "bf16").check(variant, scale=scale)
    Case(6, [33, 1], [150, 200], 4, 2, 64, 16, "fp16", spread=4.0).check(variant, scale=scale)
    Case(7, [33, 1], [150, 200], 4, 2, 64, 16, "bf16", "e4m3").check(variant, scale=scale)


@pytest.mark.parametrize("power", [-90, -20, 17, 100])
def test_bf16_queries_out_of_float16_range_over_codes(power):
    """bfloat16 queries far from 1 over an e4m3 cache, whose products run in float16: the softmax scale brings the
    logits back, and rows of one tile differ in range."""
    c = Case(30, [40, 1], [150, 300], 4, 2, 64, 16, "bf16", "e4m3")
    c.q *= 2.0 ** power
    c.check(2, scale=0.125 * 2.0 ** -power)
    c.q[::3] *= 2.0 ** 8
    c.q[1::3] = 0
    c.check(2, scale=0.01 * 2.0 ** -power)


@pytest.mark.parametrize("dt,cache", [("bf16", "bf16"), ("bf16", "e4m3"), ("fp16", "fp16")])
def test_kernels_agree(dt, cache):
    """Many heads, row tiles and key tiles: the two kernels within twice the roundings of P and the output."""
    c = Case(31, [700, 1, 300, 4], [3000, 5000, 300, 900], 8, 2, 128, 16, dt, cache)
    a, la = c.run(return_lse=True, _variant=1)
    b, lb = c.run(return_lse=True, _variant=2)
    half = torch.finfo(DT[dt]).eps / 2
    # each side: half a step of P and one of the result, relative to averages of |v| below 1.2 (values N(0, 1))
    assert (a.float() - b.float()).abs().max() <= 2 * (half * 1.2 + half * a.float().abs().max()) + 2 ** -14
    assert (la - lb).abs().max() <= 2 ** -14


@pytest.mark.parametrize("dt,cache", [("bf16", "bf16"), ("bf16", "e4m3")])
def test_joint_cache_and_strided_queries(dt, cache):
    """Caches that are views of one tensor, and queries that are a view of a fused projection."""
    c = Case(9, [60, 1, 5], [100, 300, 77], 4, 2, 128, 16, dt, cache, joint=True)
    wide = torch.zeros((c.q.shape[0], 8, 128), dtype=c.q.dtype, device="cuda")
    wide[:, :4] = c.q
    c.q = wide[:, :4]
    c.check(0)


def test_int64_lengths_and_rows_behind_the_last_request():
    """int64 seq_lens; query rows that no request owns keep what `out` held."""
    c = Case(11, [20, 3], [50, 70], 4, 2, 64, 16, "bf16", tail=9)
    c.lens = c.lens.long()
    out = torch.full_like(c.q, 7.0)
    assert c.check(0, out=out) is out
    assert (out[23:] == 7.0).all()


def test_long_cache_with_few_rows():
    """One decoding request on 30000 tokens: the context is split over many CTAs and joined."""
    Case(12, [1], [30000], 8, 2, 64, 16, "bf16").check(0)
    Case(13, [1, 2], [9000, 17], 8, 2, 128, 16, "bf16", "e4m3").check(0)


def test_many_requests():
    """More requests than a block has threads."""
    rng = seeded(4)
    n = 700
    contexts = rng.integers(0, 60, n)
    chunks = np.minimum(rng.integers(0, 4, n), np.maximum(contexts, 1))
    Case(14, chunks.tolist(), contexts.tolist(), 4, 2, 64, 16, "bf16").check(0)
    Case(15, chunks.tolist(), contexts.tolist(), 2, 1, 32, 16, "fp32").check(0)


@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("bs,scale", [(16, None), (4, -0.1), (128, 0.0)])
def test_few_rows_between_long_chunks_over_codes(dt, bs, scale):
    """Items of up to 16 rows go past the tensor-memory chains and share their buffers with what runs before and after."""
    chunks = [1, 300, 2, 1, 40, 65, 3, 300, 4, 1, 0, 1, 5, 257, 2]
    contexts = [1000, 700, 2, 129, 41, 1300, 128, 301, 2000, 127, 60, 0, 3, 900, 4097]
    Case(13, chunks, contexts, 8, 2, 128, bs, dt, "e4m3").check(2, scale=scale)


@pytest.mark.parametrize("seed,group", [(14, 4), (15, 1), (16, 8)])
def test_few_and_many_rows_in_turn_over_codes(seed, group):
    """Several items of every kind in each CTA, in random order: whoever skips an item meets the next one's buffers
    only when they are that one's."""
    rng = seeded(seed)
    chunks = [int(c) for c in rng.choice([1, 1, 2, 5, 20, 40, 130, 300], 240)]
    contexts = [c + int(rng.integers(0, 900)) for c in chunks]
    Case(seed, chunks, contexts, 2 * group, 2, 128, 16, "bf16", "e4m3").check(2)


@pytest.mark.parametrize("tokens", [1, 2, 40])
def test_many_short_requests_over_codes_keep_their_row_scales(tokens):
    """Short items follow one another in a CTA faster than their softmax; each row has a scale of its own."""
    rng = seeded(12 + tokens)
    contexts = [int(c) for c in rng.integers(tokens, 140, 900)]
    c = Case(11, [tokens] * 900, contexts, 8, 2, 128, 16, "bf16", "e4m3")
    power = torch.from_numpy(rng.integers(-14, 3, c.q.shape[:2]).astype(np.float32)).cuda()
    c.q = c.q * torch.exp2(power)[..., None].to(c.q.dtype)      # exact
    c.check(2)


def test_offsets_past_32_bits():
    """A cache of more than 2^31 elements whose pages lie at its end."""
    nb, bs, h, d = 17000, 16, 64, 128
    kc = torch.zeros((nb, bs, h, d), dtype=torch.float8_e4m3fn, device="cuda")
    rng = seeded(3)
    codes = numerics.e4m3_encode(rng.standard_normal((2, 2, bs, h, d)).astype(np.float32).clip(-448, 448))
    vc = torch.zeros_like(kc)
    kc.view(torch.uint8)[-2:] = dev(codes[0])
    vc.view(torch.uint8)[-2:] = dev(codes[1])
    q = dev(rng.standard_normal((3, h, d)).astype(np.float32), torch.bfloat16)
    one = torch.ones(h, device="cuda")
    bt = torch.tensor([[nb - 1, nb - 2]], dtype=torch.int32, device="cuda")
    out = _ops().paged_prefill_attention(q, kc, vc, torch.tensor([0, 3], dtype=torch.int32, device="cuda"),
                                         torch.tensor([29], dtype=torch.int32, device="cuda"), bt, k_scale=one, v_scale=one)
    val = numerics.e4m3_decode(codes).astype(np.float64)
    ref, _, weight, reach = attention.paged_prefill_attention(host(q), val[0], val[1], [0, 3], [29], [[1, 0]], d ** -0.5)
    bound = 2.0 ** -8 * np.abs(ref) + (2.0 ** -8 + 2 * reach[..., None] * d * 2.0 ** -23 + 2.0 ** -16) * weight
    assert (np.abs(host(out) - ref) <= bound * 1.01).all()


def test_bad_pages_and_requests_are_flagged():
    """A block-table entry out of range counts as zeros and sets bit 1; a request whose lengths do not fit
    is skipped and sets bit 2; the other requests come out as ever."""
    from kernelverse_b200 import _lib
    c = Case(16, [10, 20, 5], [40, 64, 30], 4, 2, 64, 16, "bf16")
    want = c.run()
    assert _lib.lib().kvb_device_status(1) == 0
    good = c.bt.clone()
    for entry in (-1, 1 << 30):
        c.bt[1, 2] = entry
        got = c.run()
        assert _lib.lib().kvb_device_status(1) == 2
        assert torch.equal(got[:10], want[:10]) and torch.equal(got[30:], want[30:]) and got.isfinite().all()
        c.bt.copy_(good)
    for lens in ([40, -1, 30], [40, 1 << 20, 30]):
        c.lens.copy_(torch.tensor(lens, dtype=torch.int32))
        out = torch.full_like(c.q, 3.0)
        c.run(out=out)
        assert _lib.lib().kvb_device_status(1) == 4
        assert torch.equal(out[:10], want[:10]) and torch.equal(out[30:], want[30:]) and (out[10:30] == 3.0).all()
    c.lens.copy_(torch.tensor([40, 64, 30], dtype=torch.int32))
    c.qo.copy_(torch.tensor([0, 10, 30, 36], dtype=torch.int32))              # past the last row
    got = c.run()
    assert _lib.lib().kvb_device_status(1) == 4 and torch.equal(got[:30], want[:30])
    c.qo.copy_(torch.tensor([-2, 10, 30, 35], dtype=torch.int32))
    got = c.run()
    assert _lib.lib().kvb_device_status(1) == 4 and torch.equal(got[10:], want[10:])


def test_refusals():
    c = Case(17, [4], [20], 4, 2, 64, 16, "bf16")
    ops = _ops()
    call = lambda **kw: ops.paged_prefill_attention(**dict(  # noqa: E731
        dict(q=c.q, k_cache=c.kc, v_cache=c.vc, qo_indptr=c.qo, seq_lens=c.lens, block_table=c.bt), **kw))
    with pytest.raises(TypeError, match="int32"):
        call(qo_indptr=c.qo.long())
    with pytest.raises(TypeError, match="int32"):
        call(block_table=c.bt.long())
    with pytest.raises(ValueError, match="qo_indptr"):
        call(seq_lens=c.lens.repeat(2))
    with pytest.raises(TypeError, match="e4m3"):
        call(k_cache=c.kc.half(), v_cache=c.vc.half())
    with pytest.raises(ValueError, match="caches"):
        call(v_cache=c.vc[:-1])
    with pytest.raises(ValueError, match="scales"):
        call(k_scale=torch.ones(2, device="cuda"), v_scale=torch.ones(2, device="cuda"))
    with pytest.raises(ValueError, match="one entry"):
        call(k_cache=c.kc.to(torch.float8_e4m3fn), v_cache=c.vc.to(torch.float8_e4m3fn), k_scale=torch.ones(3, device="cuda"),
             v_scale=torch.ones(3, device="cuda"))
    with pytest.raises(ValueError, match="out must be"):
        call(out=torch.empty((4, 4, 64), device="cuda"))
    with pytest.raises(RuntimeError, match="max_seq_len"):
        call(max_seq_len=10000)
    with pytest.raises(RuntimeError, match="num_q_heads"):
        call(q=torch.zeros((4, 3, 64), dtype=torch.bfloat16, device="cuda"))
    with pytest.raises(RuntimeError, match="not finite"):
        call(scale=float("nan"))


def test_equal_inputs_give_equal_outputs_and_streams_do_not_share():
    """Two streams at once on different inputs, several times: always the bits of a call alone."""
    a = Case(18, [1, 300, 2], [5000, 300, 900], 8, 2, 128, 16, "bf16")
    b = Case(19, [7, 1, 90], [800, 6000, 400], 8, 2, 128, 16, "bf16", "e4m3")
    wa, wb = a.run(return_lse=True), b.run(return_lse=True)
    torch.cuda.synchronize()
    sa, sb = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(5):
        with torch.cuda.stream(sa):
            ga = a.run(return_lse=True)
        with torch.cuda.stream(sb):
            gb = b.run(return_lse=True)
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(ga + gb, wa + wb))


def test_captured_graphs_replay_on_changed_lengths():
    """Two captured calls with one set of buffers: replayed after the lengths and queries change, both give
    what eager calls give (no length is read on the host)."""
    c = Case(20, [6, 30, 1], [400, 90, 2500], 8, 2, 128, 16, "bf16")
    c.run()
    torch.cuda.synchronize()
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        o1 = c.run()
    with torch.cuda.graph(g2):
        o2 = c.run(scale=0.3)
    c.lens.copy_(torch.tensor([350, 33, 2100], dtype=torch.int32))
    c.qo.copy_(torch.tensor([0, 30, 36, 37], dtype=torch.int32))
    c.q.neg_()
    g1.replay()
    g2.replay()
    torch.cuda.synchronize()
    assert torch.equal(o1, c.run()) and torch.equal(o2, c.run(scale=0.3))


@pytest.mark.parametrize("dt,cache", [("bf16", "bf16"), ("bf16", "e4m3"), ("fp32", "fp32")])
def test_append_then_attend(dt, cache):
    """The serving sequence: a prompt in two chunks, then two decoded tokens, each appended (normalised,
    rotated, at its position) and attended from the paged cache, next to a second request of other lengths.
    At every step the result is the oracle's attention over the cache as it stands, and the cache holds the
    oracle's keys."""
    ops, rng = _ops(), seeded(21)
    hq, hkv, d, bs = 8, 2, 64, 16
    table = ops.rope_cos_sin(512, d, device="cuda")
    qw, kw = (dev((1 + 0.1 * rng.standard_normal(d)).astype(np.float32), DT[dt]) for _ in range(2))
    ks = vs = None
    if cache == "e4m3":
        ks, vs = (torch.full((hkv,), s, device="cuda") for s in (0.02, 0.015))
    shape = (24, bs, hkv, d)
    kc = torch.zeros(shape, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn) if ks is not None else \
        torch.zeros(shape, dtype=DT[dt], device="cuda")
    vc = kc.clone()
    bt = dev(rng.permutation(24).astype(np.int32).reshape(2, 12))
    have = [0, 0]
    for chunks in ([100, 17], [41, 1], [1, 1], [1, 1]):
        t = sum(chunks)
        x = dev(rng.standard_normal((t, (hq + 2 * hkv) * d)).astype(np.float32), DT[dt])
        q, k, v = (x[:, i:j].view(t, -1, d) for i, j in ((0, hq * d), (hq * d, (hq + hkv) * d), ((hq + hkv) * d, x.shape[1])))
        pos = np.concatenate([h + np.arange(n) for h, n in zip(have, chunks)])
        req = np.repeat([0, 1], chunks)
        slots = host(bt)[req, pos // bs].astype(np.int64) * bs + pos % bs
        qr = ops.rope_paged_kv_append(q, k, v, kc, vc, dev(slots), dev(pos), table, ks, vs, qw, kw)
        have = [h + n for h, n in zip(have, chunks)]
        qo = np.concatenate([[0], np.cumsum(chunks)]).astype(np.int32)
        out = ops.paged_prefill_attention(qr, kc, vc, dev(qo), dev(np.array(have, np.int32)), bt, k_scale=ks, v_scale=vs)
        kref, size = rope.norm_rope(host(k), host(kw), pos, host(table), 1e-6, False)
        step = 2.0 ** -4 if ks is not None else torch.finfo(DT[dt]).eps / 2
        val = lambda c, s: (numerics.e4m3_decode(host(c)).astype(np.float64) * host(s)[None, None, :, None] if s is not None  # noqa: E731
                            else host(c).astype(np.float64))
        kv, vv = val(kc, ks), val(vc, vs)
        got = kv.reshape(-1, hkv, d)[slots]
        floor = 2.0 ** -10 * 0.02 if ks is not None else 0.0
        assert (np.abs(got - kref) <= np.maximum(step * np.abs(kref), floor) + 2.0 ** -18 * size).all()
        ref, _, weight, reach = attention.paged_prefill_attention(host(qr), kv, vv, qo, have, host(bt), d ** -0.5)
        half = torch.finfo(DT[dt]).eps / 2
        bound = half * np.abs(ref) + ((2.0 ** -21 if dt == "fp32" else half) + 2 * reach[..., None] * (d * 2.0 ** -23 + 2.0 ** -21)
                                      + 2.0 ** -16) * weight
        assert (np.abs(host(out) - ref) <= bound * 1.01).all()


@pytest.mark.parametrize("bs", [16, 128])
def test_few_rows_right_after_wide_items_over_codes(bs):
    """Wide items whose last key tile only the lower half of their rows sees, each followed by items of few rows that
    wrap around the ring of copies: the groups part at different tiles of the one and start the other together."""
    rng = seeded(40 + bs)
    chunks, contexts = [], []
    for _ in range(250):
        n = int(rng.integers(34, 65))                        # 4 heads: 136 to 256 rows
        chunks += [n, 1]
        contexts += [128 * int(rng.integers(1, 6)) + max(1, n - 40), int(rng.integers(129, 900))]
    Case(41, chunks, contexts, 8, 2, 128, bs, "bf16", "e4m3").check(2)


@pytest.mark.parametrize("dt,d", [("bf16", 128), ("fp16", 64)])
def test_items_whose_last_tile_one_chain_leaves_out(dt, d):
    """Wide items whose upper rows, and deep ones whose upper keys, end a tile early, in turn and followed by items that
    wrap around the ring: each chain's issuer keeps step with the copies."""
    rng = seeded(42 + d)
    chunks, contexts = [], []
    for _ in range(150):
        n = int(rng.integers(34, 65))
        chunks += [n, int(rng.integers(1, 30)), 1]
        contexts += [128 * int(rng.integers(1, 6)) + max(1, n - 40), 128 * int(rng.integers(1, 6)) + int(rng.integers(1, 65)),
                     int(rng.integers(30, 900))]
    Case(43, chunks, contexts, 8, 2, d, 16, dt).check(2)


@pytest.mark.parametrize("cache", ["bf16", "e4m3"])
def test_launches_longer_than_the_wait_limit(cache):
    """The limit of a wait is for one hand-over, not for a CTA's whole share.  A long prompt whose page tail comes last
    (16-bit caches), and wide items behind many of few rows (codes), with the limit far below the launch's duration."""
    from kernelverse_b200 import _lib
    ops, d, hkv, bs = _ops(), 128, 8, 16
    chunks, contexts = ([49151], [49151]) if cache == "bf16" else ([1] * 600 + [64, 64], [65536] * 600 + [300, 300])
    g = torch.Generator(device="cuda").manual_seed(1)
    pages = -(-max(contexts) // bs)
    kv = torch.randn((pages, 2, bs, hkv, d), generator=g, device="cuda")
    kv = kv.to(torch.bfloat16 if cache == "bf16" else torch.float8_e4m3fn)
    one = None if cache == "bf16" else torch.ones(hkv, device="cuda")
    q = torch.randn((sum(chunks), 32, d), generator=g, device="cuda").to(torch.bfloat16)
    bt = torch.arange(pages, dtype=torch.int32, device="cuda").expand(len(chunks), pages)       # shared pages
    qo = dev(np.concatenate([[0], np.cumsum(chunks)]).astype(np.int32))
    lens = dev(np.array(contexts, np.int32))
    run = lambda: ops.paged_prefill_attention(q, kv[:, 0], kv[:, 1], qo, lens, bt, k_scale=one, v_scale=one, _variant=2)  # noqa: E731
    want = run()
    begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    assert _lib.lib().kvb_device_status(1) == 0
    try:
        _lib.call("kvb_set_wait_limit_ns", 2_000_000)
        begin.record()
        got = run()
        end.record()
        assert _lib.lib().kvb_device_status(1) == 0
    finally:
        _lib.call("kvb_set_wait_limit_ns", 0)
    assert begin.elapsed_time(end) > 6.0                     # ms: what the test is about
    assert torch.equal(got, want)
