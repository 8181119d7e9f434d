"""Attention over the 4-bit cache where rows differ widely in size: large rows that weigh nothing, small ones that
carry the result, rows of zeros with all the weight, large keys among small ones.

Tolerance, per output channel of group g. A row's values are codes' part and middle,
s (c - 7.5) + (z + 7.5 s), so a row adds terms of at most m_tg = 7.5 s_tg + |z_tg + 7.5 s_tg|. A score is
off by at most delta_t = 2 gamma_(d+16) scale * sum|q||k_t| (tests/test_kv4.py), which moves a weight by
a relative delta_t + sum_s p_s delta_s, and sums of n terms add 2 (n + 32) u:
    sum_t p_t m_tg (delta_t + sum_s p_s delta_s + 2 (n + 32) u).
What carries nothing, p_t m_tg near 0, adds nothing to that bound, however large its values are. Where the
groups of a row differ, what a group may lose to the 16-bit range of an operand is 2^-24 of the largest
group's part: m_tg is taken at least 2^-12 max_g m_tg in the u term's place, 2^-12 of 2^-12.
"""
import math

import numpy as np
import pytest
import torch

from test_kv4 import GROUP, U, dev, pack, quantise

HEADS, HEADS_Q = 2, 6
FORMS = [False, True]  # single tokens, a block of positions


def stored(ctx, k, v):
    """A cache of one sequence holding k and v, f32 [n, heads, d], and the f64 values and parameters."""
    from shardlm_b200.kv4 import Kv4Cache

    n, heads, d = k.shape
    cap = -(-n // 16) * 16 + 32
    t, out = [], []
    for x, keys in ((k, True), (v, False)):
        codes = np.random.default_rng(n).integers(0, 256, (1, heads, cap, d // 2), dtype=np.uint8)
        params = np.full((1, heads, cap, 2, d // GROUP), np.nan, np.float16)
        c, p, val = quantise(x.astype(np.float32))
        codes[0, :, :n], params[0, :, :n] = np.swapaxes(pack(c, keys), 0, 1), np.swapaxes(p, 0, 1)
        t += [dev(codes), dev(params)]
        out.append((val.astype(np.float64), p.astype(np.float64)))
    return Kv4Cache.from_tensors(ctx, *t), out


def expect(q, k, v, v_params):
    """One head: q [d], k and v [n, d], v_params [n, 2, groups], all f64 -> (output [d], tolerance [d])."""
    n, d = k.shape
    scale = 1 / math.sqrt(d)
    s = (k @ q) * scale
    p = np.exp(s - s.max())
    p /= p.sum()
    delta = 2 * (d + 16) * U * scale * (np.abs(k) @ np.abs(q))
    sc, z = v_params[:, 0], v_params[:, 1]
    m = 7.5 * sc + np.abs(z + 7.5 * sc)
    m_all = np.maximum(m, m.max(-1, keepdims=True) * 2.0 ** -12)
    tol = p @ (m * (delta + p @ delta)[:, None]) + 2 * (n + 32) * U * (p @ m_all)
    return p @ v, np.repeat(tol, GROUP) + 1e-37


def run(ctx, k, v, q, prompt):
    """The last rows of the sequence (q [rows, heads_q * d]) against the expectation."""
    cache, ((kx, _), (vx, vp)) = stored(ctx, k, v)
    n, rows, d = k.shape[0], q.shape[0], k.shape[2]
    heads_q = q.shape[1] // d
    if prompt:
        got, _ = cache.attend_prompt(dev(q), slot=0, pos0=n - rows)
    else:
        got, _ = cache.attend(dev(q), slot=dev(np.zeros(rows, np.int32)), pos=dev(np.arange(n - rows, n).astype(np.int32)))
    ctx.sync()
    got = got.double().cpu().numpy().reshape(rows, heads_q, d)
    for r in range(rows):
        for h in range(heads_q):
            kv, e = h // (heads_q // HEADS), n - rows + r + 1
            want, tol = expect(q[r].reshape(heads_q, d)[h].astype(np.float64), kx[:e, kv], vx[:e, kv], vp[:e, kv])
            off = np.abs(got[r, h] - want) / tol
            assert np.all(off <= 1.0), (r, h, float(off.max()))


def direction(rng, d):
    u = rng.choice([-1.0, 1.0], (HEADS, d)) * rng.uniform(0.5, 1.5, (HEADS, d))
    return u / np.linalg.norm(u, axis=-1, keepdims=True)


def queries(rng, u, rows, along=6.0):
    """Every head some way along its kv head's direction, and noise."""
    d = u.shape[1]
    q = 0.3 * rng.standard_normal((rows, HEADS_Q, d)) + along * rng.uniform(1, 2, (rows, HEADS_Q, 1)) * np.repeat(u, HEADS_Q // HEADS, 0)
    return q.reshape(rows, -1).astype(np.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("prompt", FORMS)
@pytest.mark.parametrize("small", [1.0, 1e-3, 1e-5, 4e-7])
@pytest.mark.parametrize("at", [(40,), (0, 31, 100, 170), tuple(range(0, 192, 9))])
def test_large_rows_that_weigh_nothing(ctx, d, prompt, small, at):
    """Values of 4000 in rows whose keys point away from the queries, all others small."""
    rng = np.random.default_rng(len(at) + d)
    n, u = 200, direction(rng, d)
    k, v = rng.standard_normal((n, HEADS, d)), small * rng.standard_normal((n, HEADS, d))
    at = list(at)
    k[at] = -400.0 * u
    v[at] = 4000.0 * rng.uniform(-1, 1, (len(at), HEADS, d))
    run(ctx, k, v, queries(rng, u, 5), prompt)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("prompt", FORMS)
@pytest.mark.parametrize("first", [0.0, 1e-6, 1e-3, 1.0])
@pytest.mark.parametrize("gap", [10.0, 25.0])
def test_first_rows_with_most_of_the_weight_and_small_values(ctx, d, prompt, first, gap):
    """Two first rows that take all but e^-gap of the weight and add little or nothing."""
    rng = np.random.default_rng(int(gap) + d)
    n, u = 130, direction(rng, d)
    k, v = 0.2 * rng.standard_normal((n, HEADS, d)), rng.standard_normal((n, HEADS, d))
    k[:2] = gap * math.sqrt(d) / 9.0 * u
    v[:2] *= first
    run(ctx, k, v, queries(rng, u, 4), prompt)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("prompt", FORMS)
def test_rows_of_every_size(ctx, d, prompt):
    """Sizes 2^-14 to 2^14 in random order under scores that spread as widely the other way."""
    rng = np.random.default_rng(d)
    n, u = 256, direction(rng, d)
    e = rng.integers(-14, 15, n)
    k, v = 0.2 * rng.standard_normal((n, HEADS, d)), rng.standard_normal((n, HEADS, d)) * 2.0 ** e[:, None, None]
    k += (-e * math.log(2.0) * math.sqrt(d) / 9.0)[:, None, None] * u
    run(ctx, k, v, queries(rng, u, 6), prompt)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("prompt", FORMS)
def test_large_rows_far_apart(ctx, d, prompt):
    """A sequence that is cut into parts, with large rows that weigh nothing in a few of them."""
    rng = np.random.default_rng(d + 1)
    n, u = 2700, direction(rng, d)
    k, v = rng.standard_normal((n, HEADS, d)), 1e-5 * rng.standard_normal((n, HEADS, d))
    at = [3, 700, 1409, 2100, 2690]
    k[at], v[at] = -400.0 * u, 4000.0
    v[at[1]] = 0.0
    run(ctx, k, v, queries(rng, u, 12), prompt)


@pytest.mark.gpu
@pytest.mark.parametrize("prompt", FORMS)
def test_groups_of_different_size(ctx, prompt):
    """Groups of a row up to 2^10 apart, which ones differing from row to row, beside large rows without weight."""
    rng = np.random.default_rng(7)
    n, d = 150, 128
    u = direction(rng, d)
    e = rng.integers(-10, 1, (n, HEADS, d // GROUP))
    k, v = rng.standard_normal((n, HEADS, d)), rng.standard_normal((n, HEADS, d)) * np.repeat(2.0 ** e, GROUP, -1)
    k[33] = -400.0 * u
    v[33] = 4000.0
    run(ctx, k, v, queries(rng, u, 5), prompt)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("prompt", FORMS)
@pytest.mark.parametrize("zeros", [False, True])
def test_large_keys_among_small_ones(ctx, d, prompt, zeros):
    """Keys of 6e4 away from the queries, the others small enough that the queries make up for it."""
    rng = np.random.default_rng(d + zeros)
    n, u = 140, direction(rng, d)
    k, v = 1e-4 * rng.standard_normal((n, HEADS, d)), rng.standard_normal((n, HEADS, d))
    if zeros:
        k[::3] = 0.0
    k[[5, 77]] = -6e4 * u * math.sqrt(d) / 2
    q = queries(rng, u, 5, along=20.0) * np.float32(300.0)
    run(ctx, k, v, q, prompt)


@pytest.mark.gpu
@pytest.mark.parametrize("prompt", FORMS)
@pytest.mark.parametrize("size", [1e-30, 1e6, 1e8, 1e9, 3e9, 1e10, 3e10, 1e11, 3e11, 1e12, 1e13, 1e22, 1e30, 2e35])
def test_queries_of_any_size(ctx, prompt, size):
    """Queries over f32's range, scores to match, under values of every size: results stay finite and are those
    of the largest score where f32 can tell scores apart."""
    rng = np.random.default_rng(11)
    n, d = 100, 64
    u = direction(rng, d)
    k = rng.standard_normal((n, HEADS, d)) * (1e-4 if size > 1 else 1e3)
    v = rng.standard_normal((n, HEADS, d)) * 2.0 ** rng.integers(-12, 13, (n, HEADS, 1))
    q = (queries(rng, u, 4) * size).astype(np.float32)
    run(ctx, k, v, q, prompt)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("prompt", FORMS)
@pytest.mark.parametrize("size", [0.0, 1e-6, 1.0, 65504.0])
def test_rows_of_one_value(ctx, d, prompt, size):
    """Value rows whose channels are all alike, so that every scale is 0: alone, and half of them beside ordinary rows."""
    rng = np.random.default_rng(d + int(size))
    n, u = 90, direction(rng, d)
    k = rng.standard_normal((n, HEADS, d))
    v = np.broadcast_to(size * rng.choice([-1.0, 1.0], (n, HEADS, 1)), (n, HEADS, d)).copy()
    q = queries(rng, u, 4)
    run(ctx, k, v, q, prompt)
    v[::2] = rng.standard_normal((n // 2, HEADS, d))
    run(ctx, k, v, q, prompt)
