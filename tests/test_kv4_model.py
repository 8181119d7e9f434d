"""The model loop over a 4-bit key/value cache (shd_model_set_kv4), against the oracle's layer arithmetic
with the cache's own values: prompts, single tokens, a window with sinks over a ring, V3 and V3-MPC.

The q/k/v linear sums in another order than the oracle, so a K or V element near the middle between two
codes may round to the other one: such an element may differ by its group's step, every other one by no
more than the f32 tolerance carried through s * c + z. What is read back from the model is then what the
oracle's attention gets, and the logits are held to the model tests' tolerance.
"""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

LOGIT_RTOL = 2e-4


class OneLayer:
    """One layer of the model in the oracle's arithmetic, K and V handed in."""

    def __init__(self, orc, shape, host, max_seq, variant, mask=None):
        self.orc, self.s, self.host, self.variant, self.mask = orc, shape, host, variant, mask
        self.w = host["layers"][0]
        self.cos, self.sin = orc.rope_table(shape.head_dim, max_seq, shape.rope_theta)

    def part(self, lo, n):
        return None if self.mask is None else self.mask[lo:lo + n]

    def qkv(self, hc, hs, p):
        """Reconstructed q, k, v (RoPE applied) of position p."""
        o, s, w = self.orc, self.s, self.w
        xc, xs = o.rmsnorm_reshare(hc, hs, w["g1"], s.rms_eps, self.variant, self.part(0, s.hidden))
        out = []
        for name, bias, heads in (("wq", "bq", s.n_heads), ("wk", "bk", s.n_kv_heads), ("wv", "bv", 0)):
            c, sv = (y[0] for y in o.linear_bf16(w[name], w[bias], xc, xs))
            if heads:
                c, sv = (o.rope_apply(y, heads, s.head_dim, self.cos[p], self.sin[p]) for y in (c, sv))
            out.append(c + sv)
        return out

    def logits(self, hc, hs, p, keys, values):
        """Logits of position p, whose visible K and V rows are given."""
        o, s, w, I, h = self.orc, self.s, self.w, self.s.intermediate, self.s.hidden
        q = self.qkv(hc, hs, p)[0]
        # the softmax over the 4-bit cache is not clamped: the oracle's form without the clamp
        ac, as_ = o.attention(q, keys, values, s.n_heads, s.n_kv_heads, s.head_dim, o.NL_MPC,
                              self.part(h, s.n_heads * s.head_dim))
        dc, ds = (y[0] for y in o.linear_bf16(w["wo"], None, ac, as_))
        hc, hs = hc + dc, hs + ds
        xc, xs = o.rmsnorm_reshare(hc, hs, w["g2"], s.rms_eps, self.variant, self.part(2 * h, h))
        g, u = o.linear_bf16(w["wg"], None, xc, xs), o.linear_bf16(w["wu"], None, xc, xs)
        ac, as_ = o.swiglu_reshare(g[0][0], g[1][0], u[0][0], u[1][0], self.variant, self.part(3 * h, I))
        dc, ds = (y[0] for y in o.linear_bf16(w["wd"], None, ac, as_))
        xc, xs = o.rmsnorm_reshare(hc + dc, hs + ds, self.host["final_norm"], s.rms_eps, self.variant, self.part(0, h))
        lc, ls = o.linear_bf16(self.host["lm_head_in_out"], None, xc, xs)
        return lc[0] + ls[0]


def check_rows(x, got, d):
    """Read-back rows against the plain quantiser of tests/test_kv4.py on the oracle's f32 rows."""
    from test_kv4 import quantise

    _, params, want = quantise(x.reshape(-1, d))
    step = np.repeat(params[:, 0].astype(np.float32), 32, axis=-1)
    off = np.abs(got.reshape(-1, d) - want)
    scale = np.maximum(np.abs(x).max(), 1e-3)
    assert np.all(off <= step * 1.01 + 2e-3 * scale)
    # a differing code is a rare rounding, a parameter off by an f16 rounding a small shift
    assert np.mean(off > 2e-3 * scale) < 2e-3


def visible(p, window, sinks):
    return [t for t in range(p + 1) if not window or t < sinks or t > p - window]


@pytest.mark.parametrize("name,mpc,prompt,cap,window,sinks,max_seq", [
    ("tiny", False, 37, None, 0, 0, 64),
    ("tiny", True, 37, None, 16, 2, 64),
    ("qwen2.5-1.5b", False, 150, None, 0, 0, 176),
    ("tiny", False, 1200, 640, 100, 4, 1300),   # the sequence goes round the ring, in three prompt blocks
])
def test_model_over_4_bit_cache(ctx, orc, name, mpc, prompt, cap, window, sinks, max_seq):
    from shardlm_b200._lib import NL_MPC
    from shardlm_b200.model import SHAPES, SecureModel
    from shardlm_b200.sharing import beaver_triples_f32

    orc.set_threads(orc.max_threads())
    shape = SHAPES[name].replace(n_layers=1, vocab=1000)
    kw = dict(variant_decode=NL_MPC, variant_prefill=NL_MPC, variant_attn=NL_MPC) if mpc else {}
    m = SecureModel(ctx, shape, max_seq=max_seq, share_seed=5, **kw)
    host = m.load_random_weights(seed=11, host_copy=True)
    m.set_kv4(cap, window=window, sinks=sinks)
    mask = None
    if mpc:
        a = beaver_triples_f32(ctx, 4 * shape.hidden + 2 * shape.intermediate, seed=4).a
        m.set_masks(a[None])
        mask = a.cpu().numpy()
    ref_p = OneLayer(orc, shape, host, max_seq, orc.NL_MPC if mpc else orc.NL_GPU, mask)
    ref_d = OneLayer(orc, shape, host, max_seq, orc.NL_MPC if mpc else orc.NL_APPROX, mask)
    rng = np.random.default_rng(prompt)
    n, d = prompt + 3, shape.head_dim
    x = (rng.standard_normal((n, shape.hidden)) * 0.5).astype(np.float32)
    hs = rng.uniform(0, 1, x.shape).astype(np.float32)
    hc = (x - hs).astype(np.float32)

    def rows(p):
        """K and V of the positions that p sees, as the model holds them."""
        parts = [(0, p + 1)]
        if window:
            first = next((i for i in visible(p, window, sinks) if i >= sinks), None)
            parts = [(0, min(sinks, p + 1))] if sinks else []
            if first is not None:
                parts.append((first, p + 1 - first))
        ks, vs = zip(*[m.read_kv(a, c) for a, c in parts])
        return np.concatenate([k[0] for k in ks]), np.concatenate([v[0] for v in vs])

    _, lc, ls, _, _ = m.prefill_hidden(hc[:prompt], hs[:prompt])
    p = prompt - 1
    k, v = rows(p)
    assert k.shape[0] == len(visible(p, window, sinks))
    want = ref_p.logits(hc[p], hs[p], p, k, v)
    assert np.max(np.abs(lc + ls - want)) <= LOGIT_RTOL * np.max(np.abs(want))
    for at in sorted({p, max(0, p - 13)}):  # what the cache holds against what the layer gives
        _, kx, vx = ref_p.qkv(hc[at], hs[at], at)
        kr, vr = m.read_kv(at, 1)
        check_rows(kx, kr[0, 0], d)
        check_rows(vx, vr[0, 0], d)
    for p in range(prompt, n):
        lc, ls = m.forward_host(hc[p], hs[p])
        k, v = rows(p)
        want = ref_d.logits(hc[p], hs[p], p, k, v)
        assert np.max(np.abs(lc + ls - want)) <= LOGIT_RTOL * np.max(np.abs(want)), p
    m.close()


def test_greedy_decode_over_4_bit_cache_equals_token_by_token(ctx, orc):
    """The captured decode step of several sequences against the one-token entry on the same model."""
    from shardlm_b200.model import TINY, SecureModel

    shape, steps = TINY, 5
    prompts = [[1, 2, 3, 999, 5], [7] * 20, [400, 8]]
    tokens = {}
    for graph in (True, False):
        m = SecureModel(ctx, shape, max_seq=64, max_batch=3, share_seed=9)
        host = m.load_random_weights(seed=2, host_copy=True)
        m.set_kv4(window=12, sinks=1)
        first = [m.prefill(p, slot=i) for i, p in enumerate(prompts)]
        if graph:
            tokens[graph] = np.vstack([first, m.decode(steps, n_active=3)])
        else:
            out = [first]
            for _ in range(steps):
                nxt = []
                for i, p in enumerate(prompts):
                    pos = m.seq_len(i)
                    hc, hs = orc.embed_shares(host["embed"], shape.hidden, int(out[-1][i]), 9, (i << 32) + pos)
                    lc, ls = m.forward_host(hc, hs, slot=i)
                    nxt.append(orc.argmax_last(lc, ls))
                out.append(nxt)
            tokens[graph] = np.array(out)
        m.close()
    assert np.array_equal(tokens[True], tokens[False])


def test_set_kv4_refusals(ctx):
    from shardlm_b200._lib import SHD_ERR_ARG, ShdError
    from shardlm_b200.model import TINY, SecureModel

    m = SecureModel(ctx, TINY, max_seq=600)
    m.load_random_weights(seed=1)
    for args in ((0, 0, 0), (600, -1, 0), (600, 0, -1), (608, 0, 608), (592, 0, 0), (560, 60, 0), (560, 45, 5)):
        with pytest.raises(ShdError) as e:
            m.set_kv4(*args[:1], window=args[1], sinks=args[2])
        assert e.value.code == SHD_ERR_ARG, args
    m.set_kv4(560, window=44, sinks=5)  # 44 + 511 <= 560 - 5
    m.prefill([1, 2, 3])
    with pytest.raises(ShdError):
        m.set_kv4(600)
    k, v = m.read_kv(0, 3)
    assert np.all(np.isfinite(k)) and k.shape == (2, 3, 128)
    m.reset()
    m.set_kv4()
    assert m.prefill([1, 2, 3]) >= 0
    m.close()
