"""A sequence taken in blocks and the same sequence token by token: the caches end up bit for bit the same, and every
position's attention agrees with 64 bits in both forms, from the first token to far past a ring's capacity."""
import numpy as np
import pytest
import torch

from test_kv4 import attention64, dev, visible

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads,heads_q,d,cap,window,sinks,blocks", [
    (2, 6, 64, 96, 50, 4, [40, 1, 43, 17, 40, 43, 2, 30]),    # round the ring twice; the longest blocks it takes
    (1, 7, 128, 80, 33, 40, [8, 8, 8, 1, 5, 8, 8, 8, 8, 8, 7, 8, 8]),  # a ring no longer than the window needs
    (2, 2, 128, 224, 0, 0, [1, 15, 16, 17, 64, 100, 3]),      # everything visible, no ring
])
def test_blocks_and_single_tokens_agree(ctx, heads, heads_q, d, cap, window, sinks, blocks):
    from shardlm_b200.kv4 import Kv4Cache

    rng = np.random.default_rng(cap)
    n = sum(blocks)
    k, v = (rng.standard_normal((n, heads * d)).astype(np.float32) for _ in range(2))
    q = rng.standard_normal((n, heads_q * d)).astype(np.float32)
    block, token = (Kv4Cache(ctx, 2, heads, cap, d, sinks=sinks) for _ in range(2))
    for c in (block, token):
        for t in (c.k_codes, c.v_codes):
            t.zero_()
        for t in (c.k_params, c.v_params):
            t.fill_(float("nan"))
    out = {"block": [], "token": []}
    slot = torch.ones(1, dtype=torch.int32, device="cuda")
    values = []
    p = 0
    for rows in blocks:
        at = slice(p, p + rows)
        values.append(block.write_prompt(dev(k[at]), None, dev(v[at]), None, slot=1, pos0=p, values=True))
        out["block"].append(block.attend_prompt(dev(q[at]), slot=1, pos0=p, window=window)[0])
        for i in range(p, p + rows):
            pos = torch.full((1,), i, dtype=torch.int32, device="cuda")
            token.write(dev(k[i:i + 1]), None, dev(v[i:i + 1]), None, slot=slot, pos=pos)
            out["token"].append(token.attend(dev(q[i:i + 1]), slot=slot, pos=pos, window=window)[0])
        p += rows
        ctx.sync()
        for name in ("k_codes", "v_codes", "k_params", "v_params"):
            a, b = getattr(block, name), getattr(token, name)
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)), (p, name)
    kx, vx = (torch.cat([y[j] for y in values]).double().cpu().numpy().reshape(n, heads, d) for j in range(2))
    got = {name: torch.cat(y).double().cpu().numpy().reshape(n, heads_q, d) for name, y in out.items()}
    for i in range(n):
        t = visible(i, window, sinks)
        for h in range(heads_q):
            kv = h // (heads_q // heads)
            want, tol = attention64(q[i].reshape(heads_q, d)[h].astype(np.float64), kx[t, kv], vx[t, kv])
            for name in got:
                assert np.all(np.abs(got[name][i, h] - want) <= tol), (name, i, h)
