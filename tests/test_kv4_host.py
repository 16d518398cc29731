"""Refusals of the 4-bit key/value cache, on a machine without a GPU: the pool,
the wrappers' checks (which run before anything touches the device) and the C
entries' own."""

import ctypes
from types import SimpleNamespace

import pytest
import torch

from forgeml_b200 import _native
from forgeml_b200.nebula import CacheError, DecoderConfig, Engine, KV4Pool, KVCache, ParallelContext, ops
from oracle import kv4 as orc

EINVAL, EUNSUPPORTED = 1, 2
F32, F16, BF16 = _native.FML_F32, _native.FML_F16, _native.FML_BF16
FAKE = 1 << 20  # aligned, never dereferenced
CPU = torch.device("cpu")


@pytest.mark.parametrize("bad,match", [
    (dict(slots=0), "slots must be a positive integer"),
    (dict(heads=True), "heads must be a positive integer"),
    (dict(max_seq_len=-1), "max_seq_len must be a positive integer"),
    (dict(head_dim=2.0), "head_dim must be a positive integer"),
    (dict(head_dim=257), "head_dim <= 256"),
    (dict(dtype=torch.float64), "not supported"),
    (dict(device=CPU), "needs a CUDA device"),
    (dict(slots=1 << 64), "too large"),
    (dict(heads=1 << 19), "too large"),
    (dict(slots=1 << 30, heads=1 << 18, max_seq_len=1 << 30), "too large"),  # would wrap round 64 bits
])
def test_pool_refusals(bad, match):
    kw = dict(slots=1, heads=1, max_seq_len=8, head_dim=64, device=torch.device("cuda", 0), dtype=torch.bfloat16)
    with pytest.raises(CacheError, match=match):
        KV4Pool(**{**kw, **bad})


@pytest.mark.parametrize("bits", [8, 0, True, "4", 4.0])
def test_cache_and_engine_take_4_bits_or_none(bits):
    with pytest.raises(CacheError, match="kv_bits"):
        KVCache(layer_ids=(0,), num_heads=1, head_dim=8, max_seq_len=8, max_requests=1, device=CPU,
                dtype=torch.float32, kv_bits=bits)
    with pytest.raises(ValueError, match="kv_bits"):
        Engine(DecoderConfig(), context=ParallelContext.from_env(device="cpu"), kv_bits=bits)


def test_a_quantised_cache_needs_cuda():
    with pytest.raises(CacheError, match="CUDA"):
        KVCache(layer_ids=(0,), num_heads=1, head_dim=8, max_seq_len=8, max_requests=1, device=CPU,
                dtype=torch.float32, kv_bits=4)
    with pytest.raises(ValueError, match="requires CUDA"):
        Engine(DecoderConfig(), context=ParallelContext.from_env(device="cpu"), kv_bits=4)


def fake_pool(**kw):
    return SimpleNamespace(**{**dict(device=CPU, dtype=torch.bfloat16, heads=2, head_dim=64, max_seq_len=32), **kw})


def i32(*v):
    return torch.tensor(v, dtype=torch.int32)


def kv(b=2, t=3, h=2, d=64, dtype=torch.bfloat16):
    return torch.zeros(b, t, h, d, dtype=dtype)


@pytest.mark.parametrize("slots,starts,match", [
    ([0, 1], i32(0, 0), "slot_of must be"),
    (i32(0, 1).long(), i32(0, 0), "slot_of must be"),
    (i32(0, 1), i32(0, 0).long(), "start_pos must be"),
    (i32(0, 1).view(2, 1), i32(0, 0), "slot_of must be"),
    (i32(0, 7, 1, 7)[::2], i32(0, 0), "slot_of must be"),
    (i32(0, 1), i32(0), "one entry per request"),
    (i32(), i32(), "must not be empty"),
    (i32(0, 1).to("meta"), i32(0, 0), "pool's device"),
])
def test_wrappers_refuse_bad_tables(slots, starts, match):
    for call in (lambda: ops.kv4_append(kv(), kv(), fake_pool(), slots, starts),
                 lambda: ops.kv4_attention(kv(), fake_pool(), slots, starts),
                 lambda: ops.kv4_read(fake_pool(), slots, 3, start_pos=starts)):
        with pytest.raises(ValueError, match=match):
            call()


@pytest.mark.parametrize("k,v,match", [
    (kv(), None, "must be a tensor"),
    (kv()[0], kv(), "must be a tensor"),
    (kv(dtype=torch.float16), kv(), "device and dtype"),
    (kv(), kv(d=32), "bad v shape"),
    (kv(h=3), kv(h=3), "bad k shape"),
    (kv(b=3), kv(b=3), "bad k shape"),
    (kv(), kv(t=2), "bad v shape"),
    (kv(t=0), kv(t=0), "bad k shape"),
    (kv(t=33), kv(t=33), "max_seq_len"),
    (kv().transpose(2, 3).contiguous().transpose(2, 3), kv(), "unit stride"),
])
def test_append_refuses_bad_rows(k, v, match):
    with pytest.raises(ValueError, match=match):
        ops.kv4_append(k, v, fake_pool(), i32(0, 1), i32(0, 0))


@pytest.mark.parametrize("q,out,match", [
    (kv(h=3), None, "bad q shape"),
    (kv(h=0), None, "bad q shape"),
    (kv(b=1), None, "bad q shape"),
    (kv(t=0), None, "bad q shape"),
    (kv(d=32), None, "bad q shape"),
    (kv(t=40), None, "max_seq_len"),
    (kv(dtype=torch.float32), None, "device and dtype"),
    (kv(), torch.zeros(2, 3, 2, 64, dtype=torch.bfloat16), "out must be"),
    (kv(), torch.zeros(2, 3, 128), "out must be"),
    (kv(), torch.zeros(2, 3, 256, dtype=torch.bfloat16)[..., ::2], "out must be"),
])
def test_attention_refuses_bad_queries_and_out(q, out, match):
    with pytest.raises(ValueError, match=match):
        ops.kv4_attention(q, fake_pool(), i32(0, 1), i32(0, 0), out)


@pytest.mark.parametrize("count,out,match", [
    (0, None, "count must be"), (33, None, "count must be"), (True, None, "count must be"), (2.0, None, "count must be"),
    (3, (torch.zeros(2, 2, 3, 64),) * 2, "out must be"),
    (3, (torch.zeros(2, 3, 2, 64, dtype=torch.bfloat16),) * 2, "out must be"),
    (3, (torch.zeros(2, 2, 64, 3, dtype=torch.bfloat16).transpose(2, 3),) * 2, "out must be"),
])
def test_read_refuses_bad_counts_and_out(count, out, match):
    with pytest.raises(ValueError, match=match):
        ops.kv4_read(fake_pool(), i32(0, 1), count, out=out)


def test_pool_sizes():
    lib = _native.load()
    for slots, heads, seq, d in ((1, 1, 1, 1), (3, 2, 17, 80), (32, 16, 2048, 128), (2, 1, 100, 256)):
        n = slots * heads * -(-seq // 32) * 32 * -(-d // 32)  # groups of all rows: keys and values, codes and (s, z)
        assert lib.neb_kv4_pool_bytes(slots, heads, seq, d, BF16) == 2 * n * (16 + 4)
        assert lib.neb_kv4_pool_bytes(slots, heads, seq, d, F32) == 2 * n * (16 + 8)
    for bad in ((0, 1, 1, 1), (1, 0, 1, 1), (1, 1, 0, 1), (1, 1, 1, 0), (1, 1, 1, 257)):
        assert lib.neb_kv4_pool_bytes(*bad, BF16) == 0
    assert lib.neb_kv4_pool_bytes(1, 1, 1, 1, 9) == 0
    for big in ((1 << 31, 1, 1, 1), (1, 1 << 19, 1, 1), (1, 1, 1 << 31, 1), (1 << 30, 1 << 18, 1 << 30, 256)):
        assert lib.neb_kv4_pool_bytes(*big, BF16) == 0


def c_pool(**kw):
    f = dict(data=FAKE, slots=4, heads=2, max_seq=64, head_dim=64,
             dtype=BF16)
    return ctypes.byref(_native.neb_kv4_pool(**{**f, **kw}))


def _rejects(name, code, match, *args):
    with pytest.raises(_native.NativeError, match=match) as e:
        _native.call(name, *args)
    assert e.value.code == code


def test_c_entries_check_the_pool():
    s4 = _native.strides4((128, 128, 64, 1))
    for bad, code, match in ((None, EINVAL, "null pool"), (dict(dtype=7), EINVAL, "bad dtype"),
                             (dict(data=None), EINVAL, "null pointer"), (dict(slots=0), EINVAL, "positive"),
                             (dict(heads=-2), EINVAL, "positive"), (dict(max_seq=0), EINVAL, "positive"),
                             (dict(head_dim=300), EUNSUPPORTED, "head_dim > 256"),
                             (dict(max_seq=1 << 31), EUNSUPPORTED, "too large"),
                             (dict(data=FAKE + 16), EINVAL, "128-byte aligned")):
        p = None if bad is None else c_pool(**bad)
        _rejects("neb_kv4_append", code, match, FAKE, s4, FAKE, s4, p, FAKE, FAKE, 1, 1, None)
        _rejects("neb_kv4_read", code, match, p, FAKE, None, 1, FAKE, FAKE, 1, None)
        _rejects("neb_kv4_attention", code, match, FAKE, s4, p, FAKE, FAKE, FAKE, 1, 1, 2, 0.1, FAKE, 1 << 40, None)


def test_c_entries_check_their_arguments():
    s4, s5 = _native.strides4((128, 128, 64, 1)), _native.strides4((128, 128, 64, 2))
    p = c_pool()
    _rejects("neb_kv4_append", EINVAL, "null pointer", None, s4, FAKE, s4, p, FAKE, FAKE, 1, 1, None)
    _rejects("neb_kv4_append", EINVAL, "null pointer", FAKE, s4, FAKE, s4, p, FAKE, None, 1, 1, None)
    _rejects("neb_kv4_append", EINVAL, "positive", FAKE, s4, FAKE, s4, p, FAKE, FAKE, 0, 1, None)
    _rejects("neb_kv4_append", EINVAL, "positive", FAKE, s4, FAKE, s4, p, FAKE, FAKE, 1, -1, None)
    _rejects("neb_kv4_append", EUNSUPPORTED, "innermost stride", FAKE, s4, FAKE, s5, p, FAKE, FAKE, 1, 1, None)
    _rejects("neb_kv4_append", EUNSUPPORTED, "too many rows", FAKE, s4, FAKE, s4, p, FAKE, FAKE, 1, 65, None)
    _rejects("neb_kv4_append", EUNSUPPORTED, "too many rows", FAKE, s4, FAKE, s4, p, FAKE, FAKE, 1 << 25, 1, None)
    _rejects("neb_kv4_read", EINVAL, "null pointer", p, None, None, 1, FAKE, FAKE, 1, None)
    _rejects("neb_kv4_read", EINVAL, "positive", p, FAKE, None, 0, FAKE, FAKE, 1, None)
    _rejects("neb_kv4_read", EINVAL, "exceeds max_seq", p, FAKE, None, 65, FAKE, FAKE, 1, None)
    _rejects("neb_kv4_read", EUNSUPPORTED, "too many requests", p, FAKE, None, 1, FAKE, FAKE, 1 << 25, None)
    _rejects("neb_kv4_attention", EINVAL, "null pointer", FAKE, s4, p, FAKE, FAKE, None, 1, 1, 2, 0.1, FAKE, 1 << 40, None)
    _rejects("neb_kv4_attention", EINVAL, "positive", FAKE, s4, p, FAKE, FAKE, FAKE, 1, 1, 0, 0.1, FAKE, 1 << 40, None)
    _rejects("neb_kv4_attention", EINVAL, "multiple of the pool's heads", FAKE, s4, p, FAKE, FAKE, FAKE, 1, 1, 3, 0.1, FAKE, 1 << 40, None)
    _rejects("neb_kv4_attention", EUNSUPPORTED, "innermost stride", FAKE, s5, p, FAKE, FAKE, FAKE, 1, 1, 2, 0.1, FAKE, 1 << 40, None)
    for scale in (0.0, -1.0, float("inf"), float("nan")):
        _rejects("neb_kv4_attention", EINVAL, "positive and finite", FAKE, s4, p, FAKE, FAKE, FAKE, 1, 1, 2, scale, FAKE,
                 1 << 40, None)
    _rejects("neb_kv4_attention", EINVAL, "exceeds max_seq", FAKE, s4, p, FAKE, FAKE, FAKE, 1, 65, 2, 0.1, FAKE, 1 << 40, None)
    _rejects("neb_kv4_attention", EUNSUPPORTED, "too many queries", FAKE, s4, p, FAKE, FAKE, FAKE, 1 << 24, 64, 1 << 20,
             0.1, FAKE, 1 << 40, None)
    _rejects("neb_kv4_attention", 4, "workspace of", FAKE, s4, p, FAKE, FAKE, FAKE, 1, 1, 2, 0.1, None, 1 << 40, None)
    _rejects("neb_kv4_attention", 4, "workspace of", FAKE, s4, p, FAKE, FAKE, FAKE, 1, 1, 2, 0.1, FAKE, 64, None)
    _rejects("neb_kv4_attention", EINVAL, "16-byte aligned", FAKE, s4, p, FAKE, FAKE, FAKE, 1, 1, 2, 0.1, FAKE + 8,
             1 << 40, None)


def test_the_definition_on_hand_made_groups():
    """The oracle itself: constants, ties to even, the error's bound."""
    x = torch.zeros(1, 64)
    x[0, :32] = 2.5
    x[0, 32:] = torch.arange(32) % 16 * 1.0
    assert torch.equal(orc.stands_for(x), x.double())
    ties = torch.cat([torch.tensor([0.0, 15.0]), torch.arange(30) % 15 + 0.5]).view(1, 32)
    assert torch.equal(orc.stands_for(ties)[0, 2:], (torch.round(torch.arange(30) % 15 + 0.5)).double())
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        y = (torch.randn(50, 70, generator=torch.Generator().manual_seed(0)) * 3 + 40).to(dtype)
        for c0 in range(0, 70, 32):
            g = y[:, c0:c0 + 32].double()
            half = ((g.amax(1) - g.amin(1)) / 30 * (1 + 2.0 ** -8)).unsqueeze(1)
            assert ((orc.stands_for(y)[:, c0:c0 + 32] - g).abs() <= half).all()
