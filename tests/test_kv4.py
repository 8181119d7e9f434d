"""The 4-bit key/value cache against a plain 64-bit implementation of its format and its attention.

Tolerances. The format's steps are single f32 operations, so codes, parameters and read-back values
are compared bit for bit. Attention sums d products per score and n visible weights per output in
f32, in any order: a score is off by at most 2 gamma_(d+16) scale * sum|q||k| (Higham's bound; the
16 covers the two-term splitting of a tensor-core operand, 2^-22 of each product, and the group
sums), a weight by a relative 2 delta, and a weighted mean by another 2 (n + 32) u max|v|.
"""
import math

import numpy as np
import pytest
import torch

U = 2.0 ** -24
GROUP = 32


# ------------------------------------------------------------------------------------------------
# plain 64-bit implementation
# ------------------------------------------------------------------------------------------------
def quantise(x):
    """f32 [..., d] -> codes (channel order), params f16 [..., 2, d / 32], values f32."""
    f = np.float32
    x = np.where(np.isnan(x), f(0), np.clip(x, f(-65504), f(65504))).astype(f)
    g = x.reshape(*x.shape[:-1], -1, GROUP)
    lo, hi = g.min(-1), g.max(-1)
    z = lo.astype(np.float16)
    s = (np.maximum(hi - z.astype(f), f(0)) * f(1.0 / 15.0)).astype(np.float16)
    sf, zf = s.astype(f), z.astype(f)
    with np.errstate(divide="ignore"):
        r = np.where(sf > 0, f(1) / sf, f(0)).astype(f)
    c = np.clip(np.rint((g - zf[..., None]) * r[..., None]), 0, 15).astype(np.uint8)
    val = (sf[..., None].astype(np.float64) * c + zf[..., None]).astype(f)
    return c.reshape(x.shape), np.stack((s, z), -2), val.reshape(x.shape)


def pack(codes, keys):
    """Channel-order codes -> stored bytes, from the header's sentence on word and half-word order."""
    d = codes.shape[-1]
    ng, n = d // GROUP, 8 if keys else 4
    out = np.zeros((*codes.shape[:-1], d // 2), np.uint8)
    for ch in range(d):
        unit = ch % GROUP // n
        nib = (unit * ng + ch // GROUP) * n + ch % n
        out[..., nib // 2] |= codes[..., ch] << (4 * (nib % 2))
    return out


def row_of(p, cap, sinks):
    return p if p < cap else sinks + (p - sinks) % (cap - sinks)


def visible(p, window, sinks):
    return [t for t in range(p + 1) if not window or t < sinks or t > p - window]


def attention64(q, k, v):
    """One head: q [d], k and v [n, d] f64 -> (output, tolerance)."""
    d, n = q.size, k.shape[0]
    if n == 0:
        return np.zeros(d), np.zeros(d)
    scale = 1 / math.sqrt(d)
    s = (k @ q) * scale
    w = np.exp(s - s.max())
    w /= w.sum()
    delta = 2 * (d + 16) * U * scale * float((np.abs(k) @ np.abs(q)).max())
    tol = (2 * delta + 2 * (n + 32) * U) * float(np.abs(v).max()) + 1e-30
    return w @ v, tol


class Built:
    """A framework cache with its rows' f64 values by (slot, head, position)."""

    def __init__(self, ctx, rng, slots, heads, cap, d, sinks, lengths, k_gain=1.0, v_gain=None, garbage=True):
        from shardlm_b200.kv4 import Kv4Cache

        self.ctx = ctx
        self.k, self.v = {}, {}
        t = {}
        for name, keys in (("k", True), ("v", False)):
            codes = rng.integers(0, 256, (slots, heads, cap, d // 2), dtype=np.uint8)
            params = np.full((slots, heads, cap, 2, d // GROUP), np.nan if garbage else 0, np.float16)
            for s, n in enumerate(lengths):
                x = rng.standard_normal((n, heads, d)).astype(np.float32)
                if keys:
                    x = x * np.float32(k_gain)
                    x[..., 5::37] = x[..., 5::37] * 4 + 3
                elif v_gain is not None:
                    x = x * v_gain(np.arange(n)).astype(np.float32)[:, None, None]
                c, p, val = quantise(x)
                # later positions overwrite earlier ones where the ring has come round
                rows = np.array([row_of(i, cap, sinks) for i in range(n)], int)
                codes[s][:, rows] = np.swapaxes(pack(c, keys), 0, 1)
                params[s][:, rows] = np.swapaxes(p, 0, 1)
                getattr(self, name)[s] = val.astype(np.float64)
            t[name] = (torch.from_numpy(codes).cuda(), torch.from_numpy(params).cuda())
        self.cache = Kv4Cache.from_tensors(ctx, t["k"][0], t["k"][1], t["v"][0], t["v"][1], sinks=sinks)
        self.sinks = sinks

    def expect(self, q, slot, p, window, heads_q):
        d, hkv = self.cache.head_dim, self.cache.n_kv_heads
        y, tol = np.zeros((heads_q, d)), np.zeros((heads_q, 1))
        t = visible(p, window, self.sinks) if p >= 0 else []
        for h in range(heads_q):
            if not t:
                continue
            kv = h // (heads_q // hkv)
            y[h], tol[h] = attention64(q.reshape(heads_q, d)[h].astype(np.float64), self.k[slot][t, kv], self.v[slot][t, kv])
        return y, tol


def check_rows(got, built, q, slots, pos, window, heads_q, mask=None):
    c, s = (x.double().cpu().numpy() for x in got)
    d = built.cache.head_dim
    for m, (slot, p) in enumerate(zip(slots, pos)):
        y, tol = built.expect(q[m], slot, p, window, heads_q)
        mk = 0.0 if mask is None else mask[m].reshape(heads_q, d).astype(np.float64)
        assert np.array_equal(s[m].reshape(heads_q, d), np.broadcast_to(mk, (heads_q, d)))
        err = np.abs(c[m].reshape(heads_q, d) - (y - mk))
        room = tol + (0.0 if mask is None else U * (np.abs(y) + np.abs(mk)))
        assert np.all(err <= room), (m, slot, p, float((err - room).max()))


def dev(a, dtype=None):
    return torch.from_numpy(np.ascontiguousarray(a if dtype is None else a.astype(dtype))).cuda()


# ------------------------------------------------------------------------------------------------
# writing and reading
# ------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("d,heads,rows", [(128, 4, 1), (64, 2, 1), (128, 8, 37), (64, 3, 50), (128, 1, 300)])
@pytest.mark.parametrize("shares", [True, False])
def test_write_prompt_bit_exact(ctx, d, heads, rows, shares):
    from shardlm_b200.kv4 import Kv4Cache

    rng = np.random.default_rng(d + heads + rows)
    cap, sinks = 320, 5
    cache = Kv4Cache(ctx, 2, heads, cap, d, sinks=sinks)
    for t in (cache.k_codes, cache.v_codes, cache.k_params, cache.v_params):
        t.zero_()
    before = cache.k_codes.clone()
    # K and V as columns of one fused q|k|v row
    fused = rng.standard_normal((rows, 3 * heads * d)).astype(np.float32)
    server = rng.uniform(0, 1, fused.shape).astype(np.float32) if shares else np.zeros_like(fused)
    client = (fused - server).astype(np.float32)
    c, s = dev(client), dev(server)
    n = heads * d
    pos0 = 11 if rows <= 300 and rows + 11 <= cap else 0
    got = cache.write_prompt(c[:, n:2 * n], s[:, n:2 * n] if shares else None, c[:, 2 * n:], s[:, 2 * n:] if shares else None,
                             slot=1, pos0=pos0, values=True)
    ctx.sync()
    x = (client + server).astype(np.float32)
    for name, cols, keys, g in (("k", slice(n, 2 * n), True, got[0]), ("v", slice(2 * n, None), False, got[1])):
        codes, params, val = quantise(x[:, cols].reshape(rows, heads, d))
        at = [row_of(pos0 + i, cap, sinks) for i in range(rows)]
        assert np.array_equal(getattr(cache, name + "_codes")[1].cpu().numpy()[:, at], np.swapaxes(pack(codes, keys), 0, 1))
        assert np.array_equal(getattr(cache, name + "_params")[1].cpu().numpy()[:, at], np.swapaxes(params, 0, 1))
        assert np.array_equal(g.cpu().numpy(), val.reshape(rows, -1))
    assert torch.equal(cache.k_codes[0], before[0])  # the other sequence is untouched
    back = cache.read(1, pos0, rows)
    ctx.sync()
    assert torch.equal(back[0], got[0]) and torch.equal(back[1], got[1])


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128])
def test_write_special_groups_bit_exact(ctx, d):
    """Constant and zero groups, ranges whose scale is subnormal or rounds to 0, a minimum that rounds up,
    a wide range, one far value among equal ones."""
    from shardlm_b200.kv4 import Kv4Cache

    rng = np.random.default_rng(3)
    cases = [np.zeros(d), np.full(d, 3.3333), np.full(d, -1e-9), rng.uniform(0, 1e-6, d), rng.uniform(0, 2e-7, d),
             1000.3 + rng.uniform(0, 1e-3, d), rng.uniform(-65504, 65504, d), np.where(np.arange(d) % 32 == 7, 50.0, 1e-3),
             1e-7 * rng.standard_normal(d), np.linspace(-1, 1, d)]
    x = np.stack(cases).astype(np.float32)
    cache = Kv4Cache(ctx, 1, 1, 16, d)
    k, v = cache.write_prompt(dev(x), None, dev(-x), None, slot=0, pos0=0, values=True)
    ctx.sync()
    for got, y, name, keys in ((k, x, "k", True), (v, -x, "v", False)):
        codes, params, val = quantise(y[:, None])
        assert np.array_equal(got.cpu().numpy(), val[:, 0])
        assert np.array_equal(getattr(cache, name + "_codes")[0, 0, :len(x)].cpu().numpy(), pack(codes, keys)[:, 0])
        assert np.array_equal(getattr(cache, name + "_params")[0, 0, :len(x)].cpu().numpy(), params[:, 0])


@pytest.mark.gpu
def test_write_reports_values_the_format_cannot_hold(ctx):
    from shardlm_b200._lib import SHD_ERR_NUMERIC, ShdError
    from shardlm_b200.kv4 import Kv4Cache

    cache = Kv4Cache(ctx, 1, 2, 16, 64)
    x = np.ones((3, 128), np.float32)
    x[0, 3], x[1, 70], x[2, 5] = np.nan, np.inf, -1e6
    k, v = cache.write_prompt(dev(x), None, dev(np.ones_like(x)), None, slot=0, pos0=0, values=True)
    with pytest.raises(ShdError) as e:
        ctx.sync()
    assert e.value.code == SHD_ERR_NUMERIC
    ctx.sync()  # cleared
    assert np.array_equal(k.cpu().numpy().reshape(3, 2, 64), quantise(x.reshape(3, 2, 64))[2])
    assert torch.all(torch.isfinite(k)) and torch.all(v == 1)


@pytest.mark.gpu
def test_write_rows_of_sequences_skips_and_reports(ctx):
    from shardlm_b200._lib import SHD_ERR_ARG, ShdError
    from shardlm_b200.kv4 import Kv4Cache

    rng = np.random.default_rng(9)
    cap, sinks, d, heads = 32, 4, 128, 3
    cache = Kv4Cache(ctx, 4, heads, cap, d, sinks=sinks)
    for t in (cache.k_codes, cache.v_codes, cache.k_params, cache.v_params):
        t.zero_()
    slot, pos = np.array([2, 0, 1, 3], np.int32), np.array([31, -1, 32 + 28 * 3 + 5, 1000000007], np.int32)
    x = rng.standard_normal((4, heads * d)).astype(np.float32)
    k, _ = cache.write(dev(x), None, dev(x), None, slot=dev(slot), pos=dev(pos), values=True)
    ctx.sync()
    codes, _, val = quantise(x.reshape(4, heads, d))
    want = np.zeros((4, heads, cap, d // 2), np.uint8)
    for m in (0, 2, 3):
        want[slot[m], :, row_of(int(pos[m]), cap, sinks)] = pack(codes, True)[m]
    assert np.array_equal(cache.k_codes.cpu().numpy(), want)
    assert torch.all(k[1] == 0) and np.array_equal(k[0].cpu().numpy(), val[0].reshape(-1))
    # a slot outside the cache is skipped and reported
    kept = cache.k_codes.clone()
    cache.write(dev(x), None, dev(x), None, slot=dev(np.array([4, -1, 0, 0], np.int32)), pos=dev(np.array([0, 0, -5, -1], np.int32)))
    with pytest.raises(ShdError) as e:
        ctx.sync()
    assert e.value.code == SHD_ERR_ARG
    assert torch.equal(cache.k_codes, kept)


@pytest.mark.gpu
@pytest.mark.parametrize("pos0,n", [(0, 1), (7, 25), (40, 60), (300, 44)])
def test_read_through_the_ring(ctx, pos0, n):
    rng = np.random.default_rng(pos0)
    cap, sinks = 64, 3
    last = max(pos0 + n, 1)
    b = Built(ctx, rng, 2, 2, cap, 64, sinks, [5, last])
    if pos0 + n <= cap or n <= cap - sinks:
        k, v = b.cache.read(1, pos0, n)
        ctx.sync()
        assert np.array_equal(k.cpu().numpy(), b.k[1][pos0:pos0 + n].reshape(n, -1).astype(np.float32))
        assert np.array_equal(v.cpu().numpy(), b.v[1][pos0:pos0 + n].reshape(n, -1).astype(np.float32))
        only = torch.empty(n, 128, device="cuda")
        ctx.call("shd_kv4_read", b.cache._ref, 1, pos0, n, None, only.data_ptr())
        ctx.sync()
        assert torch.equal(only, v)


# ------------------------------------------------------------------------------------------------
# single tokens
# ------------------------------------------------------------------------------------------------
SHAPES = [(1, 1, 64), (4, 28, 128), (2, 12, 128), (8, 40, 128), (2, 4, 64), (3, 24, 128), (1, 12, 64), (2, 34, 128), (2, 2, 128)]


@pytest.mark.gpu
@pytest.mark.parametrize("heads,heads_q,d", SHAPES)
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (20, 3), (64, 0), (100, 17)])
def test_decode_short_and_ragged(ctx, heads, heads_q, d, window, sinks):
    rng = np.random.default_rng(heads_q + d + window)
    lengths = [1, 2, 15, 16, 17, 33, 100, 143]
    b = Built(ctx, rng, len(lengths), heads, 160, d, sinks, lengths)
    slots = [3, 0, 7, 5, 1, 2, 6, 4, 2]
    pos = [lengths[s] - 1 for s in slots]
    pos[-1] = -1  # an idle row
    q = rng.standard_normal((len(slots), heads_q * d)).astype(np.float32)
    mask = rng.uniform(-1, 1, q.shape).astype(np.float32) if window % 2 else None
    got = b.cache.attend(dev(q), slot=dev(np.array(slots, np.int32)), pos=dev(np.array(pos, np.int32)), window=window,
                         mask=None if mask is None else dev(mask))
    ctx.sync()
    check_rows(got, b, q, slots, pos, window, heads_q, mask)


@pytest.mark.gpu
@pytest.mark.parametrize("heads,heads_q,d,cap,window,sinks,lengths", [
    (2, 14, 128, 64, 60, 4, [64, 65, 70, 200, 124, 128]),   # the window fills the ring
    (1, 4, 64, 48, 1, 0, [49, 96, 97]),
    (2, 4, 64, 208, 100, 20, [500, 207, 208, 209, 327]),
    (2, 10, 128, 80, 33, 40, [1000, 39, 81]),
])
def test_decode_over_a_ring(ctx, heads, heads_q, d, cap, window, sinks, lengths):
    rng = np.random.default_rng(cap)
    b = Built(ctx, rng, len(lengths), heads, cap, d, sinks, lengths)
    slots, pos = list(range(len(lengths))), [n - 1 for n in lengths]
    q = rng.standard_normal((len(slots), heads_q * d)).astype(np.float32)
    got = b.cache.attend(dev(q), slot=dev(np.array(slots, np.int32)), pos=dev(np.array(pos, np.int32)), window=window)
    ctx.sync()
    check_rows(got, b, q, slots, pos, window, heads_q)


@pytest.mark.gpu
@pytest.mark.parametrize("heads,heads_q,d,length,window,sinks", [(1, 7, 128, 9001, 0, 0), (2, 2, 64, 5003, 0, 0), (1, 8, 128, 9001, 4099, 6)])
def test_decode_long_sequence_is_split_and_joined(ctx, heads, heads_q, d, length, window, sinks):
    rng = np.random.default_rng(length + heads_q)
    b = Built(ctx, rng, 2, heads, 9008, d, sinks, [length, 3])
    slots, pos = [0, 1], [length - 1, 2]
    q = rng.standard_normal((2, heads_q * d)).astype(np.float32)
    args = dict(slot=dev(np.array(slots, np.int32)), pos=dev(np.array(pos, np.int32)), window=window)
    got = b.cache.attend(dev(q), **args)
    again = b.cache.attend(dev(q), **args)
    ctx.sync()
    check_rows(got, b, q, slots, pos, window, heads_q)
    assert torch.equal(got[0], again[0])  # the order of the joins does not depend on timing


@pytest.mark.gpu
def test_decode_many_sequences(ctx):
    """More rows than SMs, lengths from 1 to the capacity, every query over its own sequence."""
    rng = np.random.default_rng(5)
    n, heads, heads_q, d = 200, 2, 6, 64
    lengths = [1 + (i * 37) % 96 for i in range(n)]
    b = Built(ctx, rng, n, heads, 96, d, 0, lengths)
    slots = list(rng.permutation(n))
    pos = [lengths[s] - 1 for s in slots]
    q = rng.standard_normal((n, heads_q * d)).astype(np.float32)
    got = b.cache.attend(dev(q), slot=dev(np.array(slots, np.int32)), pos=dev(np.array(pos, np.int32)))
    ctx.sync()
    check_rows(got, b, q, slots, pos, 0, heads_q)


@pytest.mark.gpu
def test_decode_rows_of_several_launches(ctx):
    """More rows than a launch takes, some of them empty, several on one sequence, each with its mask."""
    rng = np.random.default_rng(12)
    n, slots_n, heads, heads_q, d = 1100, 40, 1, 3, 64
    lengths = [1 + (i * 29) % 48 for i in range(slots_n)]
    b = Built(ctx, rng, slots_n, heads, 48, d, 2, lengths)
    slots = [int(x) for x in rng.integers(0, slots_n, n)]
    pos = [-1 if m % 97 == 5 else int(rng.integers(0, lengths[s])) for m, s in enumerate(slots)]
    q = rng.standard_normal((n, heads_q * d)).astype(np.float32)
    mask = rng.standard_normal((n, heads_q * d)).astype(np.float32)
    got = b.cache.attend(dev(q), slot=dev(np.array(slots, np.int32)), pos=dev(np.array(pos, np.int32)), window=20, mask=dev(mask))
    ctx.sync()
    check_rows(got, b, q, slots, pos, 20, heads_q, mask)


@pytest.mark.gpu
@pytest.mark.parametrize("parts_of", [1, 3])
def test_decode_long_beside_short(ctx, parts_of):
    """Items cut into many parts, joined in groups, next to items of one chunk."""
    rng = np.random.default_rng(13 + parts_of)
    heads, heads_q, d, length = 1, 5, 128, 12007
    lengths = [length - 1000 * i for i in range(parts_of)] + [1, 17, 2]
    b = Built(ctx, rng, len(lengths), heads, 12016, d, 0, lengths)
    slots, pos = list(range(len(lengths))), [n - 1 for n in lengths]
    q = rng.standard_normal((len(lengths), heads_q * d)).astype(np.float32)
    got = b.cache.attend(dev(q), slot=dev(np.array(slots, np.int32)), pos=dev(np.array(pos, np.int32)))
    ctx.sync()
    check_rows(got, b, q, slots, pos, 0, heads_q)


@pytest.mark.gpu
def test_prompt_of_several_launches(ctx):
    """More (position, head) tiles than a launch takes: the second launch's positions, masks and outputs."""
    rng = np.random.default_rng(14)
    heads, heads_q, d, n = 1, 64, 64, 4200
    b = Built(ctx, rng, 1, heads, 4208, d, 3, [n])
    q = rng.standard_normal((n, heads_q * d)).astype(np.float32)
    mask = rng.standard_normal((n, heads_q * d)).astype(np.float32)
    got = b.cache.attend_prompt(dev(q), slot=0, pos0=0, window=90, mask=dev(mask))
    ctx.sync()
    some = [0, 1, 2047, 4094, 4095, 4096, 4097, n - 1]
    check_rows((got[0][some], got[1][some]), b, q[some], [0] * len(some), some, 90, heads_q, mask[some])


@pytest.mark.gpu
@pytest.mark.parametrize("prompt", [False, True])
@pytest.mark.parametrize("k_gain,q_gain,v_gain", [
    (1.0, 0.0, None),                                  # equal weights
    (30.0, 5.0, None),                                 # scores in the thousands: one weight is nearly 1
    (1e-4, 1e4, None), (1.0, 1e-20, None), (100.0, 1e-3, None),
    (1.0, 1.0, lambda t: 2.0 ** (t % 23 - 16)),        # value scales 2^22 apart
    (1.0, 1.0, lambda t: np.where(t == 40, 3000.0, 1e-3)),
    (1.0, 1.0, lambda t: np.full(t.shape, 1e-6)),
])
def test_attention_extremes(ctx, prompt, k_gain, q_gain, v_gain):
    rng = np.random.default_rng(17)
    heads, heads_q, d, n = 2, 6, 128, 77
    b = Built(ctx, rng, 1, heads, 96, d, 0, [n], k_gain=k_gain, v_gain=v_gain)
    rows = 9 if prompt else 1
    q = (rng.standard_normal((rows, heads_q * d)) * q_gain).astype(np.float32)
    if prompt:
        got = b.cache.attend_prompt(dev(q), slot=0, pos0=n - rows)
    else:
        got = b.cache.attend(dev(q), slot=dev(np.array([0], np.int32)), pos=dev(np.array([n - 1], np.int32)))
    ctx.sync()
    check_rows(got, b, q, [0] * rows, range(n - rows, n), 0, heads_q)


@pytest.mark.gpu
@pytest.mark.parametrize("prompt", [False, True])
def test_nonfinite_query_stays_in_its_head(ctx, prompt):
    rng = np.random.default_rng(2)
    heads, heads_q, d, n = 2, 8, 64, 50
    b = Built(ctx, rng, 1, heads, 64, d, 0, [n])
    rows = 3
    q = rng.standard_normal((rows, heads_q * d)).astype(np.float32)
    bad = q.copy()
    bad[1, 2 * d + 5] = np.nan
    if prompt:
        run = lambda x: b.cache.attend_prompt(dev(x), slot=0, pos0=n - rows)[0]
    else:
        idx = dict(slot=dev(np.zeros(rows, np.int32)), pos=dev(np.full(rows, n - 1, np.int32)))
        run = lambda x: b.cache.attend(dev(x), **idx)[0]
    want, got = run(q).cpu().numpy(), run(bad).cpu().numpy()
    ctx.sync()
    hit = np.zeros_like(want, bool)
    hit[1, 2 * d:3 * d] = True
    assert np.all(np.isnan(got[hit])) and np.array_equal(got[~hit], want[~hit])


# ------------------------------------------------------------------------------------------------
# blocks of positions
# ------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("heads,heads_q,d", SHAPES)
@pytest.mark.parametrize("pos0,rows,window,sinks", [(0, 1, 0, 0), (0, 67, 0, 0), (30, 35, 16, 2), (63, 65, 0, 0), (100, 33, 40, 5), (5, 130, 1, 1)])
def test_prompt_blocks(ctx, heads, heads_q, d, pos0, rows, window, sinks):
    rng = np.random.default_rng(pos0 + rows + heads_q)
    b = Built(ctx, rng, 2, heads, 144, d, sinks, [9, pos0 + rows])
    q = rng.standard_normal((rows, heads_q * d)).astype(np.float32)
    mask = rng.uniform(-1, 1, q.shape).astype(np.float32) if rows % 2 else None
    got = b.cache.attend_prompt(dev(q), slot=1, pos0=pos0, window=window, mask=None if mask is None else dev(mask))
    ctx.sync()
    some = range(rows) if rows < 40 else sorted({0, 1, 15, 16, 17, 31, 32, rows // 2, rows - 2, rows - 1})
    c, s = got
    check_rows((c[list(some)], s[list(some)]), b, q[list(some)], [1] * len(some), [pos0 + m for m in some], window, heads_q,
               None if mask is None else mask[list(some)])


@pytest.mark.gpu
@pytest.mark.parametrize("heads,heads_q,d,cap,pos0,rows,window,sinks", [
    (2, 14, 128, 128, 250, 25, 100, 3),
    (1, 5, 64, 96, 90, 50, 40, 4),       # starts before the capacity, ends past it
    (2, 4, 64, 160, 1000, 30, 120, 8),
])
def test_prompt_over_a_ring(ctx, heads, heads_q, d, cap, pos0, rows, window, sinks):
    rng = np.random.default_rng(cap + pos0)
    b = Built(ctx, rng, 1, heads, cap, d, sinks, [pos0 + rows])
    q = rng.standard_normal((rows, heads_q * d)).astype(np.float32)
    got = b.cache.attend_prompt(dev(q), slot=0, pos0=pos0, window=window)
    ctx.sync()
    check_rows(got, b, q, [0] * rows, range(pos0, pos0 + rows), window, heads_q)


@pytest.mark.gpu
@pytest.mark.parametrize("heads,heads_q,d,length,rows,window,sinks", [(1, 7, 128, 6001, 5, 0, 0), (2, 2, 64, 3000, 300, 0, 0), (1, 6, 128, 4000, 700, 513, 4)])
def test_prompt_long(ctx, heads, heads_q, d, length, rows, window, sinks):
    rng = np.random.default_rng(length)
    b = Built(ctx, rng, 1, heads, 6016, d, sinks, [length])
    q = rng.standard_normal((rows, heads_q * d)).astype(np.float32)
    got = b.cache.attend_prompt(dev(q), slot=0, pos0=length - rows, window=window)
    again = b.cache.attend_prompt(dev(q), slot=0, pos0=length - rows, window=window)
    ctx.sync()
    some = sorted({0, rows // 3, rows - 2, rows - 1})
    check_rows((got[0][some], got[1][some]), b, q[some], [0] * len(some), [length - rows + m for m in some], window, heads_q)
    assert torch.equal(got[0], again[0])


@pytest.mark.gpu
def test_prompt_equals_its_tokens_one_by_one(ctx):
    """The block form and the single-token form see the same positions (ring, window and sinks)."""
    rng = np.random.default_rng(8)
    heads, heads_q, d, n = 2, 6, 64, 40
    b = Built(ctx, rng, 1, heads, 96, d, 4, [200])
    q = dev(rng.standard_normal((n, heads_q * d)).astype(np.float32))
    block, _ = b.cache.attend_prompt(q, slot=0, pos0=160, window=50)
    # single tokens need their own position to be the newest: only the last row is one
    one, _ = b.cache.attend(q[n - 1:], slot=dev(np.zeros(1, np.int32)), pos=dev(np.array([199], np.int32)), window=50)
    ctx.sync()
    y, tol = b.expect(q[n - 1].cpu().numpy(), 0, 199, 50, heads_q)
    assert np.all(np.abs(block[n - 1].cpu().numpy().reshape(heads_q, d) - one[0].cpu().numpy().reshape(heads_q, d)) <= 2 * tol)


# ------------------------------------------------------------------------------------------------
# memory, streams, graphs
# ------------------------------------------------------------------------------------------------
@pytest.mark.gpu
def test_offsets_past_32_bits(ctx):
    """A cache whose last rows lie past 2^31 bytes of codes (and 2^32 of K and V together)."""
    from shardlm_b200.kv4 import Kv4Cache

    rng = np.random.default_rng(1)
    heads, d, cap = 8, 128, 4_600_000
    cache = Kv4Cache(ctx, 1, heads, cap, d)
    assert cache.k_codes.numel() > 2 ** 31
    x = rng.standard_normal((40, heads * d)).astype(np.float32)
    y = rng.standard_normal((40, heads * d)).astype(np.float32)
    pos0 = cap - 60
    k, v = cache.write_prompt(dev(x), None, dev(y), None, slot=0, pos0=pos0, values=True)
    rk, rv = cache.read(0, pos0, 40)
    q = rng.standard_normal((40, heads * d)).astype(np.float32)
    p = pos0 + 39
    one = cache.attend(dev(q[39:]), slot=dev(np.zeros(1, np.int32)), pos=dev(np.array([p], np.int32)), window=30)
    block = cache.attend_prompt(dev(q[30:]), slot=0, pos0=pos0 + 30, window=30)
    ctx.sync()
    assert torch.equal(rk, k) and torch.equal(rv, v)
    kn, vn = (t.double().cpu().numpy().reshape(40, heads, d) for t in (k, v))
    for got, m in ((one[0][0], 39), (block[0][9], 39), (block[0][0], 30)):
        for h in range(heads):
            want, tol = attention64(q[m].reshape(heads, d)[h].astype(np.float64), kn[m - 29:m + 1, h], vn[m - 29:m + 1, h])
            assert np.all(np.abs(got.cpu().numpy().reshape(heads, d)[h] - want) <= tol)


@pytest.mark.gpu
def test_unaligned_and_strided_inputs(ctx):
    """Rows that are not 16-byte aligned, columns of a wider tensor, transposed storage."""
    rng = np.random.default_rng(6)
    heads, heads_q, d, n = 2, 4, 64, 30
    b = Built(ctx, rng, 1, heads, 32, d, 0, [n])
    q = rng.standard_normal((5, heads_q * d)).astype(np.float32)
    wide = torch.zeros(5, heads_q * d + 7, device="cuda")
    wide[:, 3:3 + heads_q * d] = dev(q)
    odd = torch.zeros(5 * heads_q * d + 1, device="cuda")[1:].reshape(5, -1)
    odd.copy_(dev(q))
    turned = dev(q).t().contiguous().t()
    want = b.cache.attend_prompt(dev(q), slot=0, pos0=n - 5)[0]
    for x in (wide[:, 3:3 + heads_q * d], odd, turned):
        assert torch.equal(b.cache.attend_prompt(x, slot=0, pos0=n - 5)[0], want)
    ctx.sync()
    check_rows((want, torch.zeros_like(want)), b, q, [0] * 5, range(n - 5, n), 0, heads_q)


@pytest.mark.gpu
def test_other_stream_and_graph(ctx):
    """Write and attend on a side stream, then captured once and replayed with moved positions."""
    rng = np.random.default_rng(12)
    heads, heads_q, d, n = 2, 8, 128, 70
    b = Built(ctx, rng, 2, heads, 96, d, 0, [n, n])
    q = rng.standard_normal((2, heads_q * d)).astype(np.float32)
    qd, slot = dev(q), dev(np.array([1, 0], np.int32))
    pos = dev(np.array([n - 1, 20], np.int32))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = b.cache.attend(qd, slot=slot, pos=pos)
        ctx.sync()
    check_rows(got, b, q, [1, 0], [n - 1, 20], 0, heads_q)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = b.cache.attend(qd, slot=slot, pos=pos)
    for at in ([5, 69], [33, 16]):
        pos.copy_(dev(np.array(at, np.int32)))
        g.replay()
        torch.cuda.synchronize()
        check_rows(got, b, q, [1, 0], at, 0, heads_q)
    ctx.bind_stream()
    ctx.sync()


# ------------------------------------------------------------------------------------------------
# refusals
# ------------------------------------------------------------------------------------------------
class _CpuContext:
    """Enough of a context for the argument checks, which come before any device call."""
    torch_device = torch.device("cpu")
    ptr = None

    def empty(self, *shape, dtype=torch.float32):
        return torch.empty(*shape, dtype=dtype)

    def bind_stream(self):
        raise AssertionError("the call was let through")


def test_argument_refusals_without_a_device():
    from shardlm_b200.kv4 import Kv4Cache
    from shardlm_b200.sharing import SharingError

    ctx = _CpuContext()
    for bad in (dict(slots=0), dict(n_kv_heads=0), dict(capacity=0), dict(head_dim=96), dict(sinks=32), dict(sinks=-1)):
        with pytest.raises(SharingError):
            Kv4Cache(ctx, **{**dict(slots=1, n_kv_heads=2, capacity=20, head_dim=64, sinks=0), **bad})
    c = Kv4Cache(ctx, 2, 2, 20, 64, sinks=3)
    assert c.capacity == 32 and c.kv_dim == 128
    assert c.device_bytes == 2 * 2 * 2 * 32 * (32 + 8)
    x, q = torch.zeros(3, 128), torch.zeros(3, 256)
    i = torch.zeros(3, dtype=torch.int32)
    refused = [
        lambda: c.write(x, None, x, x, slot=i, pos=i), lambda: c.write(x, None, x[:2], None, slot=i, pos=i),
        lambda: c.write(x.double(), None, x, None, slot=i, pos=i), lambda: c.write(x[:, :64], None, x, None, slot=i, pos=i),
        lambda: c.write(x, None, x, None, slot=i.long(), pos=i), lambda: c.write(x, None, x, None, slot=i[:2], pos=i),
        lambda: c.write_prompt(x[:0], None, x[:0], None, slot=0, pos0=0),
        lambda: c.read(0, 0, 0), lambda: c.attend(q[:, :200], slot=i, pos=i), lambda: c.attend(q, slot=i, pos=i[:1]),
        lambda: c.attend(q, slot=i, pos=i.float()), lambda: c.attend(q, slot=i, pos=i, mask=q[:2]),
        lambda: c.attend(q.half(), slot=i, pos=i), lambda: c.attend_prompt(q[0], slot=0, pos0=0),
        lambda: Kv4Cache.from_tensors(ctx, c.k_codes[:1], c.k_params, c.v_codes, c.v_params),
        lambda: Kv4Cache.from_tensors(ctx, c.k_codes, c.k_params.float(), c.v_codes, c.v_params),
        lambda: Kv4Cache.from_tensors(ctx, c.k_codes[:, :, :20], c.k_params, c.v_codes, c.v_params),
    ]
    for n, call in enumerate(refused):
        with pytest.raises(SharingError):
            call()
            raise AssertionError(f"refusal {n} did not happen")


@pytest.mark.gpu
def test_c_entry_refusals(ctx):
    import ctypes

    from shardlm_b200._lib import SHD_ERR_ARG, Kv4CacheC, ShdError
    from shardlm_b200.kv4 import Kv4Cache

    c = Kv4Cache(ctx, 2, 2, 64, 64, sinks=4)
    x = torch.zeros(100, 128, device="cuda")
    q, o = torch.zeros(100, 256, device="cuda"), torch.zeros(2, 100, 256, device="cuda")
    i = torch.zeros(100, dtype=torch.int32, device="cuda")
    X, Q, I, O, R = x.data_ptr(), q.data_ptr(), i.data_ptr(), o.data_ptr(), c._ref

    def cache(**kw):
        s = Kv4CacheC(*[getattr(c._c, f) for f, _ in Kv4CacheC._fields_])
        for k, v in kw.items():
            setattr(s, k, v)
        return ctypes.byref(s)

    refused = [
        ("shd_kv4_write", None, X, None, X, None, 128, None, None, 0, 0, 1, None, None),
        ("shd_kv4_write", cache(k_codes=None), X, None, X, None, 128, None, None, 0, 0, 1, None, None),
        ("shd_kv4_write", cache(capacity=60), X, None, X, None, 128, None, None, 0, 0, 1, None, None),
        ("shd_kv4_write", cache(head_dim=80), X, None, X, None, 128, None, None, 0, 0, 1, None, None),
        ("shd_kv4_write", cache(sinks=64), X, None, X, None, 128, None, None, 0, 0, 1, None, None),
        ("shd_kv4_write", cache(slots=0), X, None, X, None, 128, None, None, 0, 0, 1, None, None),
        ("shd_kv4_write", cache(v_params=c.v_params.data_ptr() + 2), X, None, X, None, 128, None, None, 0, 0, 1, None, None),
        ("shd_kv4_write", R, None, None, X, None, 128, None, None, 0, 0, 1, None, None),
        ("shd_kv4_write", R, X, X, X, None, 128, None, None, 0, 0, 1, None, None),
        ("shd_kv4_write", R, X, None, X, None, 128, I, None, 0, 0, 1, None, None),
        ("shd_kv4_write", R, X, None, X, None, 127, None, None, 0, 0, 1, None, None),
        ("shd_kv4_write", R, X + 4, None, X, None, 128, None, None, 0, 0, 1, None, None),
        ("shd_kv4_write", R, X, None, X, None, 128, None, None, 2, 0, 1, None, None),
        ("shd_kv4_write", R, X, None, X, None, 128, None, None, 0, -1, 1, None, None),
        ("shd_kv4_write", R, X, None, X, None, 128, None, None, 0, 0, 0, None, None),
        ("shd_kv4_write", R, X, None, X, None, 128, None, None, 0, 0, 65, None, None),
        ("shd_kv4_write", R, X, None, X, None, 128, None, None, 0, 2 ** 31 - 5, 10, None, None),
        ("shd_kv4_read", R, 2, 0, 1, O, O), ("shd_kv4_read", R, 0, 0, 0, O, O), ("shd_kv4_read", R, 0, -1, 1, O, O),
        ("shd_kv4_read", R, 0, 0, 1, None, None), ("shd_kv4_read", R, 0, 100, 61, O, O), ("shd_kv4_read", R, 0, 0, 1, O + 4, None),
        ("shd_kv4_attn_decode", R, Q, 256, 3, I, I, 1, 0, None, O, O), ("shd_kv4_attn_decode", R, None, 256, 4, I, I, 1, 0, None, O, O),
        ("shd_kv4_attn_decode", R, Q, 256, 4, I, I, 0, 0, None, O, O), ("shd_kv4_attn_decode", R, Q, 256, 4, I, I, 1, -1, None, O, O),
        ("shd_kv4_attn_decode", R, Q, 128, 4, I, I, 1, 0, None, O, O), ("shd_kv4_attn_decode", R, Q, 256, 4, None, I, 1, 0, None, O, O),
        ("shd_kv4_attn_decode", R, Q + 4, 256, 4, I, I, 1, 0, None, O, O), ("shd_kv4_attn_decode", R, Q, 256, 4, I, I, 1, 0, Q + 8, O, O),
        ("shd_kv4_attn_prefill", R, Q, 256, 4, 2, 0, 1, 0, None, O, O), ("shd_kv4_attn_prefill", R, Q, 256, 4, 0, -1, 1, 0, None, O, O),
        ("shd_kv4_attn_prefill", R, Q, 256, 4, 0, 0, 65, 0, None, O, O), ("shd_kv4_attn_prefill", R, Q, 256, 4, 0, 60, 20, 42, None, O, O),
    ]
    for n, (name, *args) in enumerate(refused):
        with pytest.raises(ShdError) as e:
            ctx.call(name, *args)
            raise AssertionError(f"refusal {n} ({name}) did not happen")
        assert e.value.code == SHD_ERR_ARG, n
    ctx.sync()


@pytest.mark.gpu
@pytest.mark.parametrize("slot,pos,window", [(2, 0, 0), (-1, 0, 0), (0, 64, 0), (0, 64, 61), (0, 2 ** 31 - 1, 0)])
def test_decode_reports_rows_the_cache_cannot_serve(ctx, slot, pos, window):
    from shardlm_b200._lib import SHD_ERR_ARG, ShdError

    rng = np.random.default_rng(4)
    b = Built(ctx, rng, 2, 2, 64, 64, 4, [64, 64])
    q = rng.standard_normal((2, 256)).astype(np.float32)
    got = b.cache.attend(dev(q), slot=dev(np.array([slot, 1], np.int32)), pos=dev(np.array([pos, 63], np.int32)), window=window)
    with pytest.raises(ShdError) as e:
        ctx.sync()
    assert e.value.code == SHD_ERR_ARG
    assert torch.all(got[0][0] == 0)
    check_rows((got[0][1:], got[1][1:]), b, q[1:], [1], [63], window, 4)
