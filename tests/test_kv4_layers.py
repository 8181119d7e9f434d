"""Models of several layers over the 4-bit cache, each layer held to the oracle with the rows that the model
holds for it: slots other than the first, mask rows at strides that are not a multiple of 16 bytes,
several sequences in one pass.

Every layer's K and V rows of a position are checked against the oracle's projections of that layer's
input, so rows of another layer or slot, which are unrelated numbers, do not pass. The bounds are those
of tests/test_kv4_model.py: an element may be off by its group's step where its code rounds the other way,
which is rare: of all elements checked (one row of 128 holds too few to say) less than 2e-3. Logits are
held to the model tests' tolerance.
"""
import numpy as np
import pytest
import torch

from test_kv4 import quantise
from test_kv4_model import LOGIT_RTOL, OneLayer, visible

pytestmark = pytest.mark.gpu


class Layers:
    """The model's layers in the oracle's arithmetic, for one position whose K and V rows are given by layer."""

    def __init__(self, orc, shape, host, max_seq, variant, masks=None):
        self.orc, self.s, self.host = orc, shape, host
        self.one = []
        for l, w in enumerate(host["layers"]):
            y = OneLayer(orc, shape, host, max_seq, variant, None if masks is None else masks[l])
            y.w = w
            self.one.append(y)

    def walk(self, hc, hs, p, keys, values):
        """(logits, [K and V of the position by layer])."""
        o, s, h, I = self.orc, self.s, self.s.hidden, self.s.intermediate
        own = []
        for l, y in enumerate(self.one):
            w = y.w
            q, k, v = y.qkv(hc, hs, p)
            own.append((k, v))
            ac, as_ = o.attention(q, keys[l], values[l], s.n_heads, s.n_kv_heads, s.head_dim, o.NL_MPC,
                                  y.part(h, s.n_heads * s.head_dim))
            dc, ds = (x[0] for x in o.linear_bf16(w["wo"], None, ac, as_))
            hc, hs = hc + dc, hs + ds
            xc, xs = o.rmsnorm_reshare(hc, hs, w["g2"], s.rms_eps, y.variant, y.part(2 * h, h))
            g, u = o.linear_bf16(w["wg"], None, xc, xs), o.linear_bf16(w["wu"], None, xc, xs)
            ac, as_ = o.swiglu_reshare(g[0][0], g[1][0], u[0][0], u[1][0], y.variant, y.part(3 * h, I))
            dc, ds = (x[0] for x in o.linear_bf16(w["wd"], None, ac, as_))
            hc, hs = hc + dc, hs + ds
        xc, xs = o.rmsnorm_reshare(hc, hs, self.host["final_norm"], s.rms_eps, y.variant, y.part(0, h))
        lc, ls = o.linear_bf16(self.host["lm_head_in_out"], None, xc, xs)
        return lc[0] + ls[0], own


def held_rows(m, slot, p, window, sinks):
    """K and V of the positions that p sees, by layer, as the model holds them."""
    t = visible(p, window, sinks)
    runs = [(t[0], 1)]
    for i in t[1:]:
        a, n = runs[-1]
        if i == a + n:
            runs[-1] = (a, n + 1)
        else:
            runs.append((i, 1))
    ks, vs = zip(*[m.read_kv(a, n, slot=slot) for a, n in runs])
    return np.concatenate(ks, 1), np.concatenate(vs, 1)


def other_codes(x, got, d):
    """Which elements of a row read back are more than the f32 tolerance off; none by more than a step."""
    _, params, want = quantise(x.reshape(-1, d))
    step = np.repeat(params[:, 0].astype(np.float32), 32, axis=-1)
    off = np.abs(got.reshape(-1, d) - want)
    scale = np.maximum(np.abs(x).max(), 1e-3)
    assert np.all(off <= step * 1.01 + 2e-3 * scale)
    return (off > 2e-3 * scale).reshape(-1)


def hidden(rng, n, h):
    x = (rng.standard_normal((n, h)) * 0.5).astype(np.float32)
    s = rng.uniform(0, 1, x.shape).astype(np.float32)
    return (x - s).astype(np.float32), s


def masks_of(ctx, shape, stride, seed):
    from shardlm_b200.sharing import beaver_triples_f32

    n = shape.n_layers * stride
    return beaver_triples_f32(ctx, n, seed=seed).a.reshape(shape.n_layers, stride)


@pytest.mark.parametrize("odd", [1, 2, 3])
@pytest.mark.parametrize("before", [True, False])
def test_mask_rows_at_any_stride(ctx, orc, odd, before):
    """Masks of three layers whose rows start anywhere, given before or after the cache is set: a prompt on
    the tensor cores, a short one, single tokens."""
    from shardlm_b200._lib import NL_MPC
    from shardlm_b200.model import TINY, SecureModel

    shape = TINY.replace(n_layers=3)
    m = SecureModel(ctx, shape, max_seq=64, max_batch=2, variant_decode=NL_MPC, variant_prefill=NL_MPC, variant_attn=NL_MPC)
    host = m.load_random_weights(seed=21, host_copy=True)
    masks = masks_of(ctx, shape, 3 * shape.hidden + shape.intermediate + odd, seed=40 + odd)
    if before:
        m.set_masks(masks)
    m.set_kv4(window=24, sinks=3)
    if not before:
        m.set_masks(masks)
    ref = Layers(orc, shape, host, 64, orc.NL_MPC, masks.cpu().numpy())
    rng = np.random.default_rng(odd)
    for slot, n in ((1, 33), (0, 2)):
        hc, hs = hidden(rng, n + 2, shape.hidden)
        _, lc, ls, _, _ = m.prefill_hidden(hc[:n], hs[:n], slot=slot)
        for p in range(n - 1, n + 2):
            if p >= n:
                lc, ls = m.forward_host(hc[p], hs[p], slot=slot)
            want, _ = ref.walk(hc[p], hs[p], p, *held_rows(m, slot, p, 24, 3))
            assert np.max(np.abs(lc + ls - want)) <= LOGIT_RTOL * np.max(np.abs(want)), (slot, p)
    m.close()


@pytest.mark.parametrize("name,window,sinks,cap", [("tiny", 0, 0, None), ("tiny", 40, 2, None), ("qwen2.5-1.5b", 0, 0, None),
                                                   ("tiny", 60, 5, 592)])
def test_every_layer_and_slot_holds_its_own_rows(ctx, orc, name, window, sinks, cap):
    """Prompts in the slots of a model of three layers, then several sequences a pass (forward_host_rows), slots out of
    order: K and V of every layer and the logits against the oracle."""
    from shardlm_b200.model import SHAPES, SecureModel

    orc.set_threads(orc.max_threads())
    shape = SHAPES[name].replace(n_layers=3, vocab=1000)
    max_seq = 80 if cap is None else 700
    m = SecureModel(ctx, shape, max_seq=max_seq, max_batch=3)
    host = m.load_random_weights(seed=3, host_copy=True)
    m.set_kv4(cap, window=window, sinks=sinks)
    prompt, token = Layers(orc, shape, host, max_seq, orc.NL_GPU), Layers(orc, shape, host, max_seq, orc.NL_APPROX)
    rng = np.random.default_rng(4)
    lengths = [23, 50 if cap is None else 610, 37]
    seqs = [hidden(rng, n + 2, shape.hidden) for n in lengths]
    differ = []

    def check(slot, p, got, ref):
        hc, hs = seqs[slot]
        want, own = ref.walk(hc[p], hs[p], p, *held_rows(m, slot, p, window, sinks))
        assert np.max(np.abs(got - want)) <= LOGIT_RTOL * np.max(np.abs(want)), (slot, p)
        k, v = m.read_kv(p, 1, slot=slot)
        for l, (kx, vx) in enumerate(own):
            differ.append(other_codes(kx, k[l, 0], shape.head_dim))
            differ.append(other_codes(vx, v[l, 0], shape.head_dim))

    for slot in (2, 0, 1):
        n = lengths[slot]
        before = [m.read_kv(0, m.seq_len(s), slot=s) for s in range(3) if s != slot and m.seq_len(s) <= 592]
        _, lc, ls, _, _ = m.prefill_hidden(seqs[slot][0][:n], seqs[slot][1][:n], slot=slot)
        check(slot, n - 1, lc + ls, prompt)
        after = [m.read_kv(0, m.seq_len(s), slot=s) for s in range(3) if s != slot and m.seq_len(s) <= 592]
        for a, b in zip(before, after):
            assert all(np.array_equal(x, y) for x, y in zip(a, b))
    for slots in ([1, 0, 2], [2, 1]):
        at = [m.seq_len(s) for s in slots]
        lc, ls = m.forward_host_rows(slots, np.stack([seqs[s][0][p] for s, p in zip(slots, at)]),
                                     np.stack([seqs[s][1][p] for s, p in zip(slots, at)]))
        for i, (s, p) in enumerate(zip(slots, at)):
            check(s, p, lc[i] + ls[i], token)
    assert np.mean(np.concatenate(differ)) < 2e-3
    m.close()


@pytest.mark.parametrize("had_kv4", [False, True])
def test_a_cache_too_large_leaves_the_model_as_it_was(ctx, had_kv4):
    """More rows than the GPU's memory: the call fails, and the model goes on with the cache it had."""
    from shardlm_b200._lib import SHD_ERR_CUDA, ShdError
    from shardlm_b200.model import TINY, SecureModel

    m = SecureModel(ctx, TINY, max_seq=64, max_batch=2)
    m.load_random_weights(seed=1)
    if had_kv4:
        m.set_kv4(window=9, sinks=2)
    want = [m.prefill([5, 6, 7, 8] * 6), *m.decode(4)[:, 0]]
    rows = m.read_kv(0, 24)
    m.reset()
    with pytest.raises(ShdError) as e:
        m.set_kv4(2 ** 31 - 16)  # 2 layers x 2 slots x 2 heads x 2^31 rows x 80 bytes and more
    assert e.value.code == SHD_ERR_CUDA
    assert [m.prefill([5, 6, 7, 8] * 6), *m.decode(4)[:, 0]] == want
    assert all(np.array_equal(a, b) for a, b in zip(rows, m.read_kv(0, 24)))
    m.close()
