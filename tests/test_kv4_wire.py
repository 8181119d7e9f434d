"""The binary wire over a 4-bit cache: a prompt that its ring cannot give back is refused before any work when the
response has to carry K and V, and taken when it has not; other responses carry what the cache holds."""
import numpy as np
import pytest

from test_wire import decode_request, parse_decode_response, parse_prefill_response, prefill_request

pytestmark = pytest.mark.gpu


def hidden(rng, n, h):
    x = (rng.standard_normal((n, h)) * 0.5).astype(np.float32)
    s = rng.uniform(0, 1, x.shape).astype(np.float32)
    return (x - s).astype(np.float32), s


@pytest.fixture(scope="module")
def ring_model(ctx):
    from shardlm_b200.model import TINY, SecureModel

    m = SecureModel(ctx, TINY.replace(n_layers=2), max_seq=1400, max_batch=2)
    m.load_random_weights(seed=6)
    m.set_kv4(640, window=100, sinks=4)  # 636 rows behind the sinks
    yield m
    m.close()


def test_prompt_longer_than_the_ring(ring_model):
    from shardlm_b200._lib import SHD_ERR_ARG, ShdError

    m = ring_model
    m.reset()
    rng = np.random.default_rng(1)
    hc, hs = hidden(rng, 700, m.shape.hidden)
    other = hidden(rng, 9, m.shape.hidden)
    m.prefill_hidden(*other, slot=1)
    kept = m.read_kv(0, 9, slot=1)
    launched = m.ctx.launch_count
    with pytest.raises(ShdError, match="ring") as e:
        m.prefill_binary(prefill_request(bytes(16), hc, hs), slot=0)
    assert e.value.code == SHD_ERR_ARG
    assert m.ctx.launch_count == launched and m.seq_len(0) == 0 and m.seq_len(1) == 9
    # a sequence that goes past the capacity by more than the ring, from where it stands
    m.prefill_binary(prefill_request(bytes(16), hc[:20], hs[:20]), slot=0)
    with pytest.raises(ShdError, match="ring"):
        m.prefill_binary(prefill_request(bytes(16), hc[:637], hs[:637]), slot=0)
    assert m.seq_len(0) == 20
    # without K and V it is taken, and the same sequence gives the same logits through the other entry
    d = parse_prefill_response(m.prefill_binary(prefill_request(bytes(16), hc[20:], hs[20:]), slot=0, include_kv=False))
    assert m.seq_len(0) == 700 and d["k_cache"].size == 0
    assert all(np.array_equal(a, b) for a, b in zip(kept, m.read_kv(0, 9, slot=1)))
    m.reset()
    m.prefill_hidden(hc[:20], hs[:20])
    _, lc, ls, fc, fs = m.prefill_hidden(hc[20:], hs[20:])
    for name, want in (("logits_client", lc), ("logits_server", ls), ("final_hidden_client", fc), ("final_hidden_server", fs)):
        assert np.array_equal(d[name], want), name


@pytest.mark.parametrize("first,n", [(0, 40), (0, 640), (4, 636), (600, 300)])
def test_responses_carry_what_the_cache_holds(ring_model, first, n):
    m = ring_model
    m.reset()
    rng = np.random.default_rng(n)
    L, h = m.shape.n_layers, m.shape.hidden
    hc, hs = hidden(rng, first + n + 1, h)
    if first:
        m.prefill_hidden(hc[:first], hs[:first], slot=1)
    d = parse_prefill_response(m.prefill_binary(prefill_request(bytes(16), hc[first:-1], hs[first:-1]), slot=1))
    k, v = m.read_kv(first, n, slot=1)
    assert np.array_equal(d["k_cache"].reshape(L, n, -1), k) and np.array_equal(d["v_cache"].reshape(L, n, -1), v)
    dd = parse_decode_response(m.decode_binary(decode_request(bytes(16), first + n, hc[-1], hs[-1]), slot=1))
    assert m.seq_len(1) == first + n + 1 and np.all(np.isfinite(dd["logits_client"]))
