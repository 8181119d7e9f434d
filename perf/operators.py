"""The 4-bit key/value cache and the attention that reads it: cases to measure, their plain forms and their 64-bit values.

Cache format. A row is one position of one kv head: head_dim channels in groups of 32. A group holds
a scale s and a minimum z (float16) and 32 codes c in 0..15, and stands for s * c + z:

    z = f16(min x)    s = f16(max(max x - z, 0) * f32(1/15))    c = clamp(rint((x - z) * (1 / s)), 0, 15)

evaluated in 32 bits (c = 0 where s = 0), x = client share + server share, NaN as 0, clamped to +-65504.
Codes are uint8 [slots][kv_heads][capacity][head_dim / 2], two a byte, even nibble low; params are
float16 [slots][kv_heads][capacity][2][head_dim / 32], scales before minima. Keys store the 8-channel
words of all groups side by side (word t of group 0, 1, .. for t = 0..3), values the 4-channel half
words (half word t of group 0, 1, .. for t = 0..7).

Position p is in row p while p < capacity; past that, rows [sinks, capacity) are a ring: position p is
in row sinks + (p - sinks) mod (capacity - sinks). A query at position p sees positions t <= p with
t < sinks or t > p - window (window 0: all).

Four operators: "write" quantises rows as they are written (single tokens of several sequences, or a
prompt) and gives the values they stand for; "read" gives rows back as f32; "decode" is attention of
one token for each of several sequences, "prompt" of a block of consecutive positions of one. Results
leave as additive shares (y - mask, mask).
"""
import math

import torch

own = False  # False: the plain forms; True: the framework's kernels

GROUP = 32
F16_MAX = 65504.0


# ------------------------------------------------------------------------------------------------
# cases
# ------------------------------------------------------------------------------------------------
def _write(name, rows, kv_heads, head_dim, capacity, prompt, sinks=0, pos0=0):
    return {"name": name, "op": "write", "rows": rows, "kv_heads": kv_heads, "head_dim": head_dim, "capacity": capacity,
            "prompt": prompt, "sinks": sinks, "pos0": pos0}


def _read(name, rows, kv_heads, head_dim, capacity, pos0=0, sinks=0):
    return {"name": name, "op": "read", "rows": rows, "kv_heads": kv_heads, "head_dim": head_dim, "capacity": capacity,
            "pos0": pos0, "sinks": sinks}


def _decode(name, seqs, kv_heads, group, head_dim, capacity, len_lo, len_hi, window=0, sinks=0, mask=False):
    return {"name": name, "op": "decode", "seqs": seqs, "kv_heads": kv_heads, "group": group, "head_dim": head_dim,
            "capacity": capacity, "len_lo": len_lo, "len_hi": len_hi, "window": window, "sinks": sinks, "mask": mask}


def _prompt(name, rows, pos0, kv_heads, group, head_dim, capacity, window=0, sinks=0, mask=False):
    return {"name": name, "op": "prompt", "rows": rows, "pos0": pos0, "kv_heads": kv_heads, "group": group,
            "head_dim": head_dim, "capacity": capacity, "window": window, "sinks": sinks, "mask": mask}


def listed():
    return [
        # one decode step of one sequence, Qwen2.5-7B heads: the smallest write
        _write("write step", 1, 4, 128, 1024, False),
        # an odd-sized prompt in head_dim 64, written past the end of a ring
        _write("write odd prompt ring", 333, 2, 64, 512, True, sinks=4, pos0=700),
        # a long prompt, Qwen2.5-14B heads
        _write("write prompt", 4096, 8, 128, 8192, True),
        # the K/V rows of a prompt response, Qwen2.5-1.5B heads
        _read("read prompt rows", 553, 2, 128, 1024, pos0=19),
        # a long sequence moved out of the cache, Qwen2.5-14B heads
        _read("read long", 32768, 8, 128, 32768),
        # the decode workload: one sequence after a 512-token prompt, Qwen2.5-7B heads
        _decode("decode one", 1, 4, 7, 128, 1024, 553, 553),
        # 8 sequences after 1024-token prompts, Qwen2.5-14B heads, masked reshare
        _decode("decode batch", 8, 8, 5, 128, 2048, 1040, 1279, mask=True),
        # one very long sequence, Qwen2.5-7B heads
        _decode("decode long", 1, 4, 7, 128, 131072, 131000, 131000),
        # many ragged streaming sequences, window and sinks over a ring, Qwen2.5-14B heads
        _decode("decode window", 64, 8, 5, 128, 2064, 17, 60000, window=2048, sinks=4),
        # the 512-token prompt, Qwen2.5-7B heads
        _prompt("prompt 512", 512, 0, 4, 7, 128, 1024),
        # a 2000-token prompt under a window with sinks, Qwen2.5-1.5B heads, masked reshare
        _prompt("prompt window", 2000, 0, 2, 6, 128, 2048, window=512, sinks=4, mask=True),
        # a prompt chunk after a long history, Qwen2.5-14B heads
        _prompt("prompt chunk", 512, 8191, 8, 5, 128, 16384),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _up16(n):
    return -(-n // 16) * 16


def draw(rng):
    op = rng.choice(["write", "read", "decode", "decode", "prompt", "prompt"])
    kv_heads, head_dim = rng.choice([1, 2, 4, 8]), rng.choice([64, 128, 128])
    case = {"op": op, "kv_heads": kv_heads, "head_dim": head_dim}
    if op == "write":
        prompt = rng.random() < 0.6
        rows = _log(rng, 1, 4096) if prompt else _log(rng, 1, 64)
        sinks = rng.choice([0, 4, 7])
        capacity = _up16(sinks + rows + _log(rng, 1, 1024))
        pos0 = rng.randrange(0, capacity - rows + 1) if rng.random() < 0.5 else _log(rng, 1, 50000)
        return {**case, "rows": rows, "capacity": capacity, "prompt": prompt, "sinks": sinks, "pos0": pos0 if prompt else 0}
    if op == "read":
        rows = _log(rng, 1, 32768)
        sinks = rng.choice([0, 4])
        return {**case, "rows": rows, "capacity": _up16(sinks + rows + _log(rng, 1, 512)), "pos0": _log(rng, 1, 2 * rows) - 1, "sinks": sinks}
    group = rng.choice([1, 2, 3, 4, 5, 6, 7, 8])
    window, sinks = (_log(rng, 1, 2048), rng.choice([0, 1, 4, 16])) if rng.random() < 0.5 else (0, 0)
    case |= {"group": group, "window": window, "sinks": sinks, "mask": rng.random() < 0.5}
    if op == "decode":
        seqs = _log(rng, 1, 64)
        len_hi = _log(rng, 1, min(65536, 131072 // seqs))
        len_lo = _log(rng, 1, len_hi)
        if window and rng.random() < 0.5:  # a ring that the sequences have gone round
            capacity = _up16(sinks + window + rng.randrange(0, 40))
        else:
            capacity = _up16(len_hi + rng.randrange(0, 200) + sinks + 1)
        return {**case, "seqs": seqs, "capacity": capacity, "len_lo": len_lo, "len_hi": len_hi}
    rows = _log(rng, 1, min(2048, math.isqrt(120_000_000 // (kv_heads * group))))
    pos0 = _log(rng, 1, max(1, min(32768, 120_000_000 // (rows * kv_heads * group) - rows))) - 1
    if window and rng.random() < 0.5:
        capacity = _up16(sinks + window + rows + rng.randrange(0, 40))
    else:
        capacity = _up16(pos0 + rows + rng.randrange(0, 200) + sinks + 1)
    return {**case, "rows": rows, "pos0": pos0, "capacity": capacity}


# ------------------------------------------------------------------------------------------------
# the plain forms
# ------------------------------------------------------------------------------------------------
def _to_order(c, keys):
    """Codes [.., head_dim] in channel order -> stored order (uint8 pairs)."""
    lead, d = c.shape[:-1], c.shape[-1]
    n = 8 if keys else 4
    c = c.reshape(*lead, d // GROUP, GROUP // n, n).transpose(-3, -2).reshape(*lead, d // 2, 2)
    return c[..., 0] | (c[..., 1] << 4)


def _from_order(packed, keys):
    """Stored codes -> uint8 codes in channel order."""
    lead, d = packed.shape[:-1], 2 * packed.shape[-1]
    n = 8 if keys else 4
    c = torch.stack((packed & 15, packed >> 4), dim=-1).reshape(*lead, GROUP // n, d // GROUP, n)
    return c.transpose(-3, -2).reshape(*lead, d)


def _quantise(x):
    """f32 [.., head_dim] -> (uint8 codes in channel order, f16 params [.., 2, groups], f32 values)."""
    lead, d = x.shape[:-1], x.shape[-1]
    x = torch.where(torch.isnan(x), torch.zeros_like(x), x).clamp(-F16_MAX, F16_MAX).reshape(*lead, d // GROUP, GROUP)
    z = x.amin(-1).half()
    zf = z.float()
    s = ((x.amax(-1) - zf).clamp_min(0.0) * torch.tensor(1.0 / 15.0, dtype=torch.float32, device=x.device)).half()
    sf = s.float()
    r = torch.where(sf > 0, 1.0 / sf, torch.zeros_like(sf))
    c = torch.round((x - zf[..., None]) * r[..., None]).clamp(0.0, 15.0)
    val = (sf[..., None] * c + zf[..., None]).reshape(*lead, d)
    return c.to(torch.uint8).reshape(*lead, d), torch.stack((s, z), dim=-2), val


def _values(packed, params, keys):
    """Stored rows -> f32 [.., head_dim]."""
    c = _from_order(packed, keys).float()
    p = params.float()
    c = c.reshape(*c.shape[:-1], c.shape[-1] // GROUP, GROUP)
    return (p[..., 0, :, None] * c + p[..., 1, :, None]).reshape(*packed.shape[:-1], -1)


def _row_of(pos, capacity, sinks):
    """Cache row of each position."""
    return torch.where(pos < capacity, pos, sinks + torch.remainder(pos - sinks, capacity - sinks))


def _visible(last, query, rows, capacity, sinks, window):
    """Which of the first `rows` cache rows a query sees, when `last` is the newest position written:
    last, query int64 [..] -> bool [.., rows]."""
    r = torch.arange(rows, device=last.device)
    last, query = last[..., None], query[..., None]
    t = torch.where(r < sinks, r, last - torch.remainder(last - r, capacity - sinks))
    seen = (t <= query) & ((r < sinks) | (t >= sinks))
    return seen & ((r < sinks) | (t > query - window)) if window else seen


def _attention(q, k, v, seen):
    """q [.., n, d], k and v [.., L, d], seen [.., n, L] -> softmax(q k^T / sqrt(d)) v, 0 where nothing is seen."""
    s = torch.matmul(q, k.transpose(-1, -2)) * (1.0 / math.sqrt(q.shape[-1]))
    s = s.masked_fill(~seen, -math.inf)
    m = s.amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(torch.isinf(m), torch.zeros_like(m), m))
    total = e.sum(-1, keepdim=True)
    return torch.matmul(e, v) / torch.where(total > 0, total, torch.ones_like(total))


def _reshare(y, mask):
    return {"c": y if mask is None else y - mask, "s": torch.zeros_like(y) if mask is None else mask.clone()}


def _plain_write(s):
    row = _row_of(s["pos"], s["capacity"], s["sinks"])
    out = {}
    for name, keys in (("k", True), ("v", False)):
        x = (s[name + "_client"] + s[name + "_server"]).reshape(-1, s["kv_heads"], s["head_dim"])
        c, p, val = _quantise(x)
        s[name + "_codes"][s["slot"], :, row] = _to_order(c, keys)
        s[name + "_params"][s["slot"], :, row] = p
        out[name] = val.reshape(val.shape[0], -1)
        out[name + "_codes"], out[name + "_params"] = s[name + "_codes"], s[name + "_params"]
    return out


def _plain_read(s):
    row = _row_of(torch.arange(s["pos0"], s["pos0"] + s["rows"], device=s["k_codes"].device), s["capacity"], s["sinks"])
    k = _values(s["k_codes"][0][:, row], s["k_params"][0][:, row], True)
    v = _values(s["v_codes"][0][:, row], s["v_params"][0][:, row], False)
    return {"k": k.transpose(0, 1).reshape(s["rows"], -1), "v": v.transpose(0, 1).reshape(s["rows"], -1)}


def _plain_decode(s):
    n, hkv, d = s["q"].shape[0], s["kv_heads"], s["head_dim"]
    seen = _visible(s["pos"], s["pos"], s["capacity"], s["capacity"], s["sinks"], s["window"])[:, None, :]  # [n, 1, rows]
    zero = torch.zeros((), device=s["q"].device)
    k = torch.where(seen[..., None], _values(s["k_codes"][s["slot"]], s["k_params"][s["slot"]], True), zero)
    v = torch.where(seen[..., None], _values(s["v_codes"][s["slot"]], s["v_params"][s["slot"]], False), zero)
    y = _attention(s["q"].reshape(n, hkv, -1, d), k, v, seen[:, :, None, :])
    return _reshare(y.reshape(n, -1), s["mask"])


def _plain_prompt(s):
    n, hkv, d = s["rows"], s["kv_heads"], s["head_dim"]
    dev = s["q"].device
    last = s["pos0"] + n - 1
    rows = min(s["capacity"], last + 1)
    seen = _visible(torch.full((n,), last, device=dev), torch.arange(s["pos0"], last + 1, device=dev), rows, s["capacity"],
                    s["sinks"], s["window"])
    some = seen.any(0)[None, :, None]
    zero = torch.zeros((), device=dev)
    k = torch.where(some, _values(s["k_codes"][s["slot0"], :, :rows], s["k_params"][s["slot0"], :, :rows], True), zero)
    v = torch.where(some, _values(s["v_codes"][s["slot0"], :, :rows], s["v_params"][s["slot0"], :, :rows], False), zero)
    q = s["q"].reshape(n, hkv, -1, d).permute(1, 2, 0, 3)  # [kv head, head of its group, row, d]
    y = _attention(q, k[:, None], v[:, None], seen[None, None])
    return _reshare(y.permute(2, 0, 1, 3).reshape(n, -1), s["mask"])


# ------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------
def _lengths(case):
    """Ragged lengths of a decode batch, spread evenly from len_lo to len_hi."""
    n, lo, hi = case["seqs"], case["len_lo"], case["len_hi"]
    return [hi if n == 1 else lo + (hi - lo) * i // (n - 1) for i in range(n)]


def _normal(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g)


def _keys(g, *shape):
    """Keys as projections give them: unit variance, a few channels of a head far larger and off zero."""
    x = _normal(g, *shape)
    x[..., 3::41] = x[..., 3::41] * 5.0 + 4.0
    return x


def _cache(case, g, slots, filled):
    """A cache of `slots` sequences, the rows listed in `filled` (positions of slot 0.. as int64 [slots][n]
    or None for all) written, the others as memory is found: any codes, any params."""
    hkv, d, cap = case["kv_heads"], case["head_dim"], case["capacity"]
    out = {}
    for name, keys in (("k", True), ("v", False)):
        codes = torch.empty(slots, hkv, cap, d // 2, dtype=torch.uint8, device="cuda")
        params = torch.empty(slots, hkv, cap, 2, d // GROUP, dtype=torch.float16, device="cuda")
        for s in range(slots):
            for r in range(0, cap, 16384):
                n = min(16384, cap - r)
                x = _keys(g, hkv, n, d) if keys else 0.5 * _normal(g, hkv, n, d)
                c, p, _ = _quantise(x)
                codes[s, :, r:r + n], params[s, :, r:r + n] = _to_order(c, keys), p
        if filled is not None:
            never = torch.arange(cap, device="cuda")[None, :] >= filled[:, None]
            params.masked_fill_(never[:, None, :, None, None], math.nan)
        out[name + "_codes"], out[name + "_params"] = codes, params
    return out


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    hkv, d, cap = case["kv_heads"], case["head_dim"], case["capacity"]
    s = {k: case[k] for k in ("op", "kv_heads", "head_dim", "capacity", "sinks")}
    if case["op"] == "write":
        n = case["rows"]
        slots = 1 if case["prompt"] else n
        s |= _cache(case, g, slots, torch.zeros(slots, dtype=torch.int64, device="cuda"))
        s |= {"prompt": case["prompt"], "pos0": case["pos0"], "slot0": 0}
        for name in ("k", "v"):
            x = _keys(g, n, hkv, d) if name == "k" else 0.5 * _normal(g, n, hkv, d)
            server = torch.rand(n, hkv * d, device="cuda", generator=g)
            s[name + "_client"], s[name + "_server"] = x.reshape(n, hkv * d) - server, server
        if case["prompt"]:
            s["slot"] = torch.zeros(n, dtype=torch.int64, device="cuda")
            s["pos"] = torch.arange(case["pos0"], case["pos0"] + n, device="cuda")
        else:
            s["slot"] = torch.randperm(n, device="cuda", generator=g)
            s["pos"] = torch.randint(0, cap, (n,), device="cuda", generator=g)
        s |= {"slot32": s["slot"].int(), "pos32": s["pos"].int()}
    elif case["op"] == "read":
        s |= _cache(case, g, 1, None)
        s |= {"rows": case["rows"], "pos0": case["pos0"], "slot0": 0}
    else:
        h = hkv * case["group"]
        s["window"] = case["window"]
        if case["op"] == "decode":
            n = case["seqs"]
            s["slot"] = torch.randperm(n, device="cuda", generator=g)
            s["pos"] = torch.tensor(_lengths(case), device="cuda")[torch.randperm(n, device="cuda", generator=g)] - 1
            held = torch.empty_like(s["pos"])
            held[s["slot"]] = s["pos"] + 1
            s |= _cache(case, g, n, held)
            s |= {"slot32": s["slot"].int(), "pos32": s["pos"].int()}
        else:
            n = case["rows"]
            s |= _cache(case, g, 2, torch.tensor([7, case["pos0"] + n], device="cuda"))
            s |= {"rows": n, "pos0": case["pos0"], "slot0": 1}
        s["q"] = _normal(g, n, h * d)
        s["mask"] = 2.0 * torch.rand(n, h * d, device="cuda", generator=g) - 1.0 if case["mask"] else None
    return s


# ------------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------------
_context = None


def _framework_cache(s):
    """The framework's cache over the state's tensors, made once as a program makes it."""
    global _context
    if "cache" not in s:
        from shardlm_b200.kv4 import Kv4Cache
        from shardlm_b200.runtime import Context

        if _context is None:
            _context = Context(torch.cuda.current_device())
        s["cache"] = Kv4Cache.from_tensors(_context, s["k_codes"], s["k_params"], s["v_codes"], s["v_params"], sinks=s["sinks"])
    return s["cache"]


def _own(s):
    cache = _framework_cache(s)
    if s["op"] == "write":
        shares = (s["k_client"], s["k_server"], s["v_client"], s["v_server"])
        if s["prompt"]:
            k, v = cache.write_prompt(*shares, slot=s["slot0"], pos0=s["pos0"], values=True)
        else:
            k, v = cache.write(*shares, slot=s["slot32"], pos=s["pos32"], values=True)
        return {"k": k, "v": v, **{n: s[n] for n in ("k_codes", "k_params", "v_codes", "v_params")}}
    if s["op"] == "read":
        k, v = cache.read(s["slot0"], s["pos0"], s["rows"])
        return {"k": k, "v": v}
    if s["op"] == "decode":
        c, sv = cache.attend(s["q"], slot=s["slot32"], pos=s["pos32"], window=s["window"], mask=s["mask"])
    else:
        c, sv = cache.attend_prompt(s["q"], slot=s["slot0"], pos0=s["pos0"], window=s["window"], mask=s["mask"])
    return {"c": c, "s": sv}


def run(state):
    if own:
        return _own(state)
    return {"write": _plain_write, "read": _plain_read, "decode": _plain_decode, "prompt": _plain_prompt}[state["op"]](state)


def _seen_positions(p, case):
    """How many positions a query at p sees."""
    if not case["window"]:
        return p + 1
    return min(p + 1, case["window"] + max(0, min(case["sinks"], p + 1 - case["window"])))


def work(case):
    hkv, d = case["kv_heads"], case["head_dim"]
    row = 2 * hkv * (d // 2 + 4 * (d // GROUP))  # K and V of one position
    if case["op"] == "write":
        n = case["rows"] * hkv * d
        return {"bytes": 16 * n + 8 * n + case["rows"] * row, "flops": 10 * n}
    if case["op"] == "read":
        n = case["rows"] * hkv * d
        return {"bytes": case["rows"] * row + 8 * n, "flops": 4 * n}
    h = hkv * case["group"]
    shares = (16 if case["mask"] else 12) * h * d  # q, mask in, two shares out
    if case["op"] == "decode":
        seen = sum(_seen_positions(n - 1, case) for n in _lengths(case))
        return {"bytes": seen * row + case["seqs"] * shares, "flops": 4 * h * d * seen}
    first, n = case["pos0"], case["rows"]
    seen = sum(_seen_positions(p, case) for p in range(first, first + n))
    reach = min(first + n, _seen_positions(first, case) + n - 1)
    return {"bytes": reach * row + n * shares, "flops": 4 * h * d * seen}


# ------------------------------------------------------------------------------------------------
# the operators' values in 64 bits
# ------------------------------------------------------------------------------------------------
def _round32(x):
    return x.float().double()


def _exact_group(x):
    """The format's definition on f64 [.., 32]: each step is one operation rounded to the bits it names."""
    lo, hi = x.min(-1).values, x.max(-1).values
    z = lo.half().double()
    s = _round32(_round32(hi - z).clamp(min=0.0) * float(torch.tensor(1.0 / 15.0, dtype=torch.float32))).half().double()
    inverse = torch.where(s > 0, _round32(1.0 / s.clamp(min=2.0 ** -30)), torch.zeros_like(s))
    c = _round32(_round32(x - z[..., None]) * inverse[..., None]).round().clamp(0, 15)
    return s, z, s[..., None] * c + z[..., None]


def _exact_rows(packed, params, keys):
    """f64 values of stored rows, channel by channel from the format's byte order."""
    d = 2 * packed.shape[-1]
    ch = torch.arange(d, device=packed.device)
    n = 8 if keys else 4
    group, unit, nibble = ch // GROUP, ch % GROUP // n, ch % n
    at = (unit * (d // GROUP) + group) * n + nibble
    byte = packed[..., at // 2].int()
    c = torch.where(at % 2 == 0, byte % 16, byte // 16).double()
    return params[..., 0, :].double()[..., group] * c + params[..., 1, :].double()[..., group]


def _exact_attend(q, k, v):
    """q [heads, d], k and v [positions, d], all f64."""
    if k.shape[0] == 0:
        return torch.zeros_like(q)
    return torch.softmax(q @ k.T / math.sqrt(q.shape[-1]), dim=-1) @ v


def _exact_row(p, case):
    cap, sinks = case["capacity"], case["sinks"]
    return p if p < cap else sinks + (p - sinks) % (cap - sinks)


def exact(case, seed):
    s = prepare(case, seed)
    hkv, d = case["kv_heads"], case["head_dim"]
    if case["op"] == "write":
        out = {}
        rows = [_exact_row(p, case) for p in s["pos"].tolist()]
        for name in ("k", "v"):
            x = _round32(s[name + "_client"].double() + s[name + "_server"].double())
            sc, z, val = _exact_group(x.reshape(-1, hkv, d // GROUP, GROUP))
            params = s[name + "_params"].double()
            params[s["slot"], :, torch.tensor(rows, device="cuda")] = torch.stack((sc, z), dim=-2)
            out[name] = val.reshape(val.shape[0], -1)
            out[name + "_codes"], out[name + "_params"] = None, params
        return out
    if case["op"] == "read":
        rows = torch.tensor([_exact_row(p, case) for p in range(case["pos0"], case["pos0"] + case["rows"])], device="cuda")
        out = {}
        for name in ("k", "v"):
            val = [_exact_rows(s[name + "_codes"][0, h, rows], s[name + "_params"][0, h, rows], name == "k") for h in range(hkv)]
            out[name] = torch.cat(val, dim=-1)
        return out
    group, window, sinks = case["group"], case["window"], case["sinks"]
    q = s["q"].double().reshape(-1, hkv, group, d)
    y = torch.zeros_like(q)
    if case["op"] == "decode":
        for i, (slot, p) in enumerate(zip(s["slot"].tolist(), s["pos"].tolist())):
            first = max(0, p - window + 1) if window else 0
            held = [_exact_row(t, case) for t in list(range(min(sinks, first))) + list(range(first, p + 1))]
            rows = torch.tensor(held, dtype=torch.int64, device="cuda")
            for h in range(hkv):
                y[i, h] = _exact_attend(q[i, h], _exact_rows(s["k_codes"][slot, h, rows], s["k_params"][slot, h, rows], True),
                                        _exact_rows(s["v_codes"][slot, h, rows], s["v_params"][slot, h, rows], False))
    else:
        p0, n = case["pos0"], case["rows"]
        first = max(0, p0 - window + 1) if window else 0
        held = list(range(min(sinks, first))) + list(range(first, p0 + n))
        rows = torch.tensor([_exact_row(t, case) for t in held], dtype=torch.int64, device="cuda")
        t = torch.tensor(held, dtype=torch.int64, device="cuda")
        for h in range(hkv):
            k = _exact_rows(s["k_codes"][1, h, rows], s["k_params"][1, h, rows], True)
            v = _exact_rows(s["v_codes"][1, h, rows], s["v_params"][1, h, rows], False)
            for i in range(0, n, 256):
                p = torch.arange(p0 + i, min(p0 + i + 256, p0 + n), device="cuda")[:, None]
                hidden = (t > p) | ((t >= sinks) & (t <= p - window)) if window else t > p
                a = torch.einsum("ngd,td->gnt", q[i:i + 256, h], k) / math.sqrt(d)
                w = torch.softmax(a.masked_fill(hidden, -math.inf), dim=-1)
                y[i:i + 256, h] = torch.einsum("gnt,td->ngd", w, v)
    y = y.reshape(y.shape[0], -1)
    mask = torch.zeros_like(y) if s["mask"] is None else s["mask"].double()
    return {"c": y - mask, "s": mask}
