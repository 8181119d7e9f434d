"""Arguments of the 4-bit cache that the C entries could not take as they are: refused, not cut to 32 bits."""
import pytest
import torch

from test_kv4 import _CpuContext

BIG = 2 ** 32


def test_integers_past_32_bits_are_refused():
    from shardlm_b200.kv4 import Kv4Cache
    from shardlm_b200.sharing import SharingError

    c = Kv4Cache(_CpuContext(), 2, 2, 32, 64, sinks=3)
    x, q = torch.zeros(3, 128), torch.zeros(3, 256)
    i = torch.zeros(3, dtype=torch.int32)
    refused = [
        lambda: c.write_prompt(x, None, x, None, slot=0, pos0=BIG), lambda: c.write_prompt(x, None, x, None, slot=BIG, pos0=0),
        lambda: c.write_prompt(x, None, x, None, slot=-BIG, pos0=0), lambda: c.read(BIG + 1, 0, 1), lambda: c.read(0, BIG, 1),
        lambda: c.read(0, 0, BIG + 1), lambda: c.attend(q, slot=i, pos=i, window=BIG),
        lambda: c.attend_prompt(q, slot=0, pos0=0, window=BIG + 5), lambda: c.attend_prompt(q, slot=BIG, pos0=0),
        lambda: c.attend_prompt(q, slot=0, pos0=BIG),
    ]
    for n, call in enumerate(refused):
        with pytest.raises(SharingError, match="32 bits"):
            call()
            raise AssertionError(f"refusal {n} did not happen")
    meta = [torch.empty(1, 1, 2 ** 31, 32, dtype=torch.uint8, device="meta"), torch.empty(1, 1, 2 ** 31, 2, 2, dtype=torch.float16, device="meta")]
    ctx = _CpuContext()
    ctx.torch_device = torch.device("meta")
    with pytest.raises(SharingError, match="32 bits"):
        Kv4Cache.from_tensors(ctx, *meta, *meta)


def test_model_arguments_past_32_bits_are_refused():
    from shardlm_b200._lib import SHD_ERR_ARG, ShdError
    from shardlm_b200.model import SecureModel

    m = SecureModel.__new__(SecureModel)  # refused before the library is asked
    m.max_seq, m.handle = 64, None
    for kw in (dict(capacity=BIG + 64), dict(window=BIG), dict(sinks=BIG), dict(window=-BIG)):
        with pytest.raises(ShdError) as e:
            m.set_kv4(**kw)
        assert e.value.code == SHD_ERR_ARG


@pytest.mark.gpu
def test_heads_whose_width_passes_32_bits_are_refused(ctx):
    """Head counts whose rows would be 2^32 channels wide, which is no width in 32 bits, at every C entry."""
    from shardlm_b200._lib import SHD_ERR_ARG, Kv4CacheC, ShdError
    from shardlm_b200.kv4 import Kv4Cache

    import ctypes

    c = Kv4Cache(ctx, 1, 2, 32, 64)
    x = torch.zeros(4, 256, device="cuda")
    i = torch.zeros(4, dtype=torch.int32, device="cuda")
    X, I, many = x.data_ptr(), i.data_ptr(), 2 ** 26
    wide = Kv4CacheC(*[getattr(c._c, f) for f, _ in Kv4CacheC._fields_])
    wide.n_kv_heads = many
    W = ctypes.byref(wide)
    for name, *args in (
        ("shd_kv4_attn_decode", c._ref, X, 256, many, I, I, 1, 0, None, X, X),
        ("shd_kv4_attn_prefill", c._ref, X, 256, many, 0, 0, 1, 0, None, X, X),
        ("shd_kv4_write", W, X, None, X, None, 256, None, None, 0, 0, 1, None, None),
        ("shd_kv4_read", W, 0, 0, 1, X, X),
        ("shd_kv4_attn_decode", W, X, 256, many, I, I, 1, 0, None, X, X),
        ("shd_kv4_attn_prefill", W, X, 256, many, 0, 0, 1, 0, None, X, X),
    ):
        with pytest.raises(ShdError) as e:
            ctx.call(name, *args)
        assert e.value.code == SHD_ERR_ARG, name
    ctx.sync()
