"""Models of several layers over the 4-bit cache, each layer held to the oracle with the rows that the model
holds for it: slots other than the first, mask rows at strides that are not a multiple of 16 bytes,
several sequences in one pass.

Every layer's K and V rows of a position are checked against the oracle's projections of that layer's
input (tests/test_kv4_model.py states what a rounding of a code may do), so rows of another layer or slot,
which are unrelated numbers, do not pass. Logits are held to the model tests' tolerance.
"""
import numpy as np
import pytest
import torch

from test_kv4_model import LOGIT_RTOL, OneLayer, check_rows, visible

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
