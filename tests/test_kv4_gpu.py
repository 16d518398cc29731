"""The 4-bit key/value cache on the B200 against its definition in float64
(oracle/kv4.py): append, read back, attention, and a run of them together.

Tolerances (u = finfo(dtype).eps / 2, one rounding to the dtype):
  read back  z + c s is formed once in fp32 and rounded to the dtype:
             (u + 2^-24) |x|, plus half the smallest subnormal.
  attention  see ``attention_bound``.
"""

import math

import pytest
import torch

from forgeml_b200 import _native
from forgeml_b200.nebula import (CacheError, DecoderConfig, Engine, KV4Pool, KVCache, ParallelContext, TinyDecoder,
                                 ops)
from oracle import kv4 as orc

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
RANGE = 4  # bit of the device error word: slot or position outside the pool


@pytest.fixture(autouse=True)
def clean_status(cuda):
    _native.device_status()
    yield
    assert _native.device_status() == 0


def rows(b, n, h, d, dtype, seed, offset=True):
    g = torch.Generator().manual_seed(seed)
    k = torch.randn(b, n, h, d, generator=g)
    if offset:
        k = k + 3.0 * torch.randn(h, d, generator=g)
    return k.to(dtype), torch.randn(b, n, h, d, generator=g).to(dtype)


def make_pool(cuda, slots, h, max_seq, d, dtype):
    pool = KV4Pool(slots=slots, heads=h, max_seq_len=max_seq, head_dim=d, device=cuda, dtype=dtype)
    pool.data.fill_(255)  # rows nobody wrote: codes 15, parameters NaN
    return pool


def table(values, cuda):
    return torch.tensor(values, dtype=torch.int32, device=cuda)


def snapshot(pool):
    """The pool's bytes: keys' codes and parameters, values' codes and parameters,
    [slots, heads, rows, bytes] each."""
    groups, es = -(-pool.head_dim // 32), torch.finfo(pool.dtype).bits // 8
    widths = [16 * groups, 2 * groups * es] * 2
    tiles = pool.data.clone().view(pool.slots, pool.heads, -1, 32 * sum(widths))
    return [x.reshape(pool.slots, pool.heads, -1, w) for x, w in zip(tiles.split([32 * w for w in widths], -1), widths)]


def check_values(got, want64, dtype):
    got = got.cpu().double()
    f = torch.finfo(dtype)
    tol = (f.eps / 2 + 2.0 ** -24) * want64.abs() + f.tiny * f.eps / 2
    assert torch.equal(got.isnan(), want64.isnan())
    bad = (got - want64).abs() > tol
    assert not bad.any(), (got[bad][:4], want64[bad][:4])


def on_tensor_cores(dtype, t, group):
    return dtype != torch.float32 and t * group > 8


def attention_bound(q, kx, vx, starts, dtype, tc):
    """float64 [B, T, QH * D]: what a kernel may be off by before the output's
    rounding.  e = 2^-24, w the weights, A = sum w |v| of an
    output, n the positions.  Weights whose scores are off by at most x are off
    by 2 x of themselves against their sum (x small), the output by 2 x A.

    Up to 8 rows of a head, or fp32 (a group of 32 channels is z + c s, its span
    15 s; a = |z| + 15 s, for fp32 |z + 8 s| + 8 s):
      scores    q as an integer q / max|q| * 1.2e8: rounded to fp32, then to the
                integer.  The products and their sums are exact; they are put
                together in fp32, (G + 8) e of scale * sum |q| a (in float64 for
                fp32).  The exponent: e times scores' distance from the maximum.
      weights   exponential 2^-22 (documented), and once more each time that the
                maximum moves, n / 32 times at the most.
      digits    p s goes as an integer, half a unit off at the most or dropped:
                min(p s, h), where 1.25 times the largest p s <= max s makes
                65530 (fp16, fp32: 8388600) units of 2 h; times 15 (the code).
      sums      of n / 32 + 40 roundings, and as many at moves of the maximum, for
                the output and for the weights: 4 (n / 32 + 40) e of sum w a.
    On the tensor cores, u = 2^-11 the rounding to fp16:
      scores    u of every |q k|, the products' fp32 sums (d + 8) 2^-23, and the
                subnormal step 2^-25 of fp16 or, scaled by powers of two to 2^12
                at least, 2^-37 of the largest |q| and |k|; the exponent as above.
      weights   2^-22 each and per move of the maximum; weights and values
                rounded, 2 u A; a weight's or value's subnormal step 2^-25 of the
                largest value; sums (n / 16 + 40) 2^-23 A."""
    b, t, qh, d = q.shape
    q = q.detach().cpu().double()
    h, n_all, u, e = kx.shape[2], kx.shape[1], 2.0 ** -11, 2.0 ** -24
    group, scale, wide = qh // h, 1 / math.sqrt(d), dtype == torch.float32
    bound = torch.empty(b, t, qh, d, dtype=torch.float64)
    kx, vx = kx.nan_to_num(0.0), vx.nan_to_num(0.0)  # rows of NaN: compared by their being NaN

    def span(x, wide):  # per number, its group's a and s
        a, st = torch.empty_like(x), torch.empty_like(x)
        for c0 in range(0, d, 32):
            g = x[..., c0:c0 + 32]
            z, s15 = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True) - g.amin(-1, keepdim=True)
            a[..., c0:c0 + 32] = ((z + s15 * 8 / 15).abs() + s15 * 8 / 15) if wide else z.abs() + s15
            st[..., c0:c0 + 32] = s15 / 15
        return a, st

    ka, _ = span(kx, False)
    va, vs = span(vx, wide)
    for i in range(b):
        n = int(starts[i]) + t
        late = torch.arange(n)[None, :] > int(starts[i]) + torch.arange(t)[:, None]
        moves = n / 32 + 1
        for hq in range(qh):
            kh, vh, qi = kx[i, :n, hq // group], vx[i, :n, hq // group], q[i, :, hq]
            sc = (qi @ kh.T * scale).masked_fill(late, -math.inf)
            w = torch.softmax(sc, -1)
            A = w @ vh.abs()
            qabs, qmax = qi.abs(), qi.abs().amax(-1, keepdim=True)
            far = (sc.amax(-1, keepdim=True) - sc).masked_fill(late, 0)
            small = qabs @ ka[i, :n, hq // group].T * scale
            if tc:
                x = (u + (d + 8) * 2 * e) * (qabs @ kh.abs().T) * scale
                if dtype == torch.float16:
                    x = x + 2.0 ** -25 * qabs.sum(-1, keepdim=True) * scale
                else:
                    x = x + 2.0 ** -37 * (qabs.sum(-1, keepdim=True) * kh.abs().max() + qmax * kh.abs().sum(-1)) * scale
                x = x + 2 * e * (far + sc.masked_fill(late, 0).abs())
                rel = moves / 4 * 2.0 ** -22 + 2.0 ** -22 + x
                vmax, top = vh.abs().max(), w.amax(-1, keepdim=True)
                other = 2 * u * A + 2.0 ** -25 * vmax * (2 + n * top) + (n / 16 + 40) * 2 * e * A
            else:
                x = e * qabs @ ka[i, :n, hq // group].T * scale + 0.6 / 1.2e8 * qmax * scale * ka[i, :n, hq // group].sum(-1)
                x = x + e * far + (0 if wide else (-(-d // 32) + 8) * e * small)
                rel = x + moves * 2.0 ** -22
                s = vs[i, :n, hq // group]
                top = w.amax(-1, keepdim=True)
                half = 0.625 * s.amax(0) / (65530 if dtype == torch.bfloat16 else 8388600)
                p = w / top  # of the largest weight
                other = 15 * top * torch.stack([torch.minimum(p[j][:, None] * s, half).sum(0) for j in range(t)])
                other = other + 4 * (n / 32 + 40) * e * (w @ va[i, :n, hq // group])
            rel = rel.masked_fill(late, 0)
            bound[i, :, hq] = (w * torch.expm1(rel)) @ vh.abs() + (w * torch.expm1(rel)).sum(-1, keepdim=True) * A + other
    return bound.reshape(b, t, qh * d)


def check_attention(got, q, kx, vx, starts, dtype, t=None):
    """t: the call's tokens, where q holds only its first ones."""
    want = orc.attention(q, kx, vx, starts)
    tc = on_tensor_cores(dtype, t or q.shape[1], q.shape[2] // kx.shape[2])
    bound = attention_bound(q, kx, vx, starts, dtype, tc)
    f = torch.finfo(dtype)
    tol = bound * (1 + f.eps) + f.eps / 2 * want.nan_to_num(0.0).abs() + f.tiny * f.eps / 2
    got = got.cpu().double()
    assert torch.equal(got.isnan(), want.isnan())
    err = (got - want).abs().masked_fill(want.isnan(), 0)
    assert (err <= tol).all(), (float((err - tol).max()), float(err.max()), float((err / tol).max()))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,t,h,d", [(1, 1, 1, 1), (2, 3, 2, 32), (3, 1, 16, 128), (2, 17, 3, 80), (1, 130, 2, 64),
                                     (2, 5, 5, 33), (1, 9, 1, 256), (2, 4, 3, 192), (1, 7, 2, 96), (1, 5, 2, 160),
                                     (2, 2, 2, 224), (1, 3, 1, 255)])
def test_rows_read_back_as_their_definition(cuda, dtype, b, t, h, d):
    k, v = rows(b, t, h, d, dtype, seed=7 * d + t)
    max_seq = t + 21
    pool = make_pool(cuda, b + 2, h, max_seq, d, dtype)
    before = snapshot(pool)
    slots = table([(3 * i + 1) % (b + 2) for i in range(b)] if (b + 2) % 3 else list(range(b, 0, -1)), cuda)
    starts = table([(5 * i + 4) % 22 for i in range(b)], cuda)
    ops.kv4_append(k.to(cuda), v.to(cuda), pool, slots, starts)
    kr, vr = ops.kv4_read(pool, slots, t, start_pos=starts)
    check_values(kr, orc.stands_for(k).transpose(1, 2), dtype)
    check_values(vr, orc.stands_for(v).transpose(1, 2), dtype)
    # every row not written is as it was
    written = torch.zeros(b + 2, max_seq + (-max_seq) % 32, dtype=torch.bool, device=cuda)
    for i in range(b):
        written[int(slots[i]), int(starts[i]):int(starts[i]) + t] = True
    keep = ~written[:, None].expand(-1, h, -1)
    for x, y in zip(before, snapshot(pool)):
        assert torch.equal(x[keep], y[keep])
    # from row 0, and into given tensors
    n = int(starts.min()) + t
    out = tuple(torch.empty(b, h, n, d, dtype=dtype, device=cuda) for _ in range(2))
    assert ops.kv4_read(pool, slots, n, out=out)[0] is out[0]
    for i in range(b):
        if n > int(starts[i]):
            torch.testing.assert_close(out[1][i, :, int(starts[i]):], vr[i, :, :n - int(starts[i])], rtol=0, atol=0)


@pytest.mark.parametrize("dtype", DTYPES)
def test_groups_at_the_borders(cuda, dtype):
    """Constant groups, ties, the type's extremes, subnormals, infinities, NaN."""
    f = torch.finfo(dtype)
    d = 64
    k = torch.zeros(1, 10, 1, d, dtype=torch.float64)
    k[0, 0] = 3.0  # constant: step 0
    k[0, 1, 0] = torch.arange(d) % 32 * 0.5  # 0 .. 15.5: ties at every half
    k[0, 2, 0] = torch.arange(d) % 16 * f.tiny * f.eps  # subnormals
    k[0, 3, 0, 0], k[0, 3, 0, 1] = f.max, f.min  # the widest range
    k[0, 4, 0] = torch.linspace(1000, 1001, d)  # far from zero
    k[0, 5, 0, 3] = math.inf
    k[0, 6, 0, 40] = math.nan
    k[0, 7, 0, 5], k[0, 7, 0, 45] = -math.inf, math.nan
    k[0, 8, 0] = torch.arange(d) % 31 * f.tiny
    k[0, 9, 0] = torch.linspace(-1, 1, d) ** 3 * math.sqrt(f.max)
    k = k.to(dtype)
    v = k.flip(1)
    pool = make_pool(cuda, 1, 1, 12, d, dtype)
    z = table([0], cuda)
    ops.kv4_append(k.to(cuda), v.to(cuda), pool, z, z)
    kr, vr = ops.kv4_read(pool, z, 10)
    check_values(kr, orc.stands_for(k).transpose(1, 2), dtype)
    check_values(vr, orc.stands_for(v).transpose(1, 2), dtype)


@pytest.mark.parametrize("dtype", DTYPES)
def test_append_from_strided_views(cuda, dtype):
    """k and v as column views of one projection output, rows that are not
    16-byte aligned, and a permuted batch."""
    b, t, h, d = 2, 5, 3, 40
    g = torch.Generator().manual_seed(3)
    for off, width in ((0, 3 * h * d), (1, 3 * h * d + 3)):
        wide = torch.randn(b * t, width, generator=g).to(dtype)
        dev = wide.to(cuda)

        def views(w):
            return [w[:, off + i * h * d:off + (i + 1) * h * d].reshape(b, t, h, d) if not w.is_cuda
                    else w[:, off + i * h * d:off + (i + 1) * h * d].unflatten(1, (h, d)).unflatten(0, (b, t))
                    for i in (1, 2)]

        pool = make_pool(cuda, 3, h, 16, d, dtype)
        slots, starts = table([2, 0], cuda), table([0, 3], cuda)
        ops.kv4_append(*views(dev), pool, slots, starts)
        kr, vr = ops.kv4_read(pool, slots, t, start_pos=starts)
        kc, vc = views(wide)
        check_values(kr, orc.stands_for(kc).transpose(1, 2), dtype)
        check_values(vr, orc.stands_for(vc).transpose(1, 2), dtype)
        # [B, H, T, D] storage seen as [B, T, H, D]
        perm = kc.transpose(1, 2).contiguous().to(cuda).transpose(1, 2)
        ops.kv4_append(perm, perm, pool, slots, starts)
        check_values(ops.kv4_read(pool, slots, t, start_pos=starts)[0], orc.stands_for(kc).transpose(1, 2), dtype)


def fill(cuda, dtype, starts, t, h, d, seed, extra_rows=5):
    """A pool holding each request's rows 0..start+t-1 (nothing behind them),
    and the same rows in float64 [B, n, H, D]."""
    b, n = len(starts), max(starts) + t
    k, v = rows(b, n, h, d, dtype, seed)
    pool = make_pool(cuda, b + 1, h, n + extra_rows, d, dtype)
    slots = [(i + 1) % (b + 1) for i in range(b)]
    for i, s in enumerate(starts):
        m = s + t
        ops.kv4_append(k[i:i + 1, :m].to(cuda), v[i:i + 1, :m].to(cuda), pool, table([slots[i]], cuda),
                       table([0], cuda))
    return pool, table(slots, cuda), table(starts, cuda), orc.stands_for(k), orc.stands_for(v)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("starts,t,h,group,d", [
    ([0], 1, 1, 1, 128),
    ([0, 1, 15, 16], 1, 2, 1, 128),
    ([17, 63, 64, 127, 128, 129], 1, 3, 1, 64),
    ([300, 5], 1, 4, 1, 80),
    ([1023, 700, 0], 1, 2, 1, 128),
    ([100, 31], 1, 2, 1, 32),
    ([100, 131], 1, 2, 1, 256),
    ([70, 9], 1, 3, 1, 96),
    ([40, 90], 1, 1, 1, 192),
    ([33], 1, 1, 1, 160),
    ([64, 12], 1, 1, 1, 224),
    ([50], 1, 2, 1, 7),
    ([200, 3], 1, 2, 4, 128),
    ([77, 150], 1, 2, 7, 64),
    ([90], 1, 1, 8, 256),
    ([33, 0, 120], 3, 2, 1, 128),
    ([140, 61], 5, 2, 2, 64),
    ([30], 2, 1, 3, 96),
])
def test_attention(cuda, dtype, starts, t, h, group, d):
    pool, slots, st, kx, vx = fill(cuda, dtype, starts, t, h, d, seed=d + t + h)
    q = torch.randn(len(starts), t, h * group, d, generator=torch.Generator().manual_seed(d)).to(dtype)
    got = ops.kv4_attention(q.to(cuda), pool, slots, st)
    assert got.shape == (len(starts), t, h * group * d)
    check_attention(got, q, kx, vx, starts, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("starts,t,h,group,d", [([0], 130, 1, 1, 128), ([0, 60], 129, 2, 1, 64), ([200], 33, 1, 2, 128),
                                                ([1, 0, 255], 40, 1, 1, 80), ([127, 128], 64, 1, 1, 128),
                                                ([5], 70, 1, 1, 256)])
def test_attention_of_prompts(cuda, dtype, starts, t, h, group, d):
    pool, slots, st, kx, vx = fill(cuda, dtype, starts, t, h, d, seed=d + t)
    q = torch.randn(len(starts), t, h * group, d, generator=torch.Generator().manual_seed(t)).to(dtype)
    got = ops.kv4_attention(q.to(cuda), pool, slots, st)
    check_attention(got, q, kx, vx, starts, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("t,d", [(1, 128), (1, 80), (4, 64), (40, 128)])
def test_attention_of_sharp_scores_and_far_keys(cuda, dtype, t, d):
    """Scores of tens whose maximum keeps moving along the rows, and channels
    far from zero."""
    starts = [611]
    n = starts[0] + t
    g = torch.Generator().manual_seed(5)
    k = torch.randn(1, n, 2, d, generator=g) + 20.0 * (torch.rand(2, d, generator=g) > 0.9)
    k = (k * torch.linspace(0.2, 1.5, n)[None, :, None, None]).to(dtype)
    v = (torch.randn(1, n, 2, d, generator=g) * 1e-2 + 1.0).to(dtype)
    pool = make_pool(cuda, 1, 2, n, d, dtype)
    z = table([0], cuda)
    ops.kv4_append(k.to(cuda), v.to(cuda), pool, z, z)
    q = (torch.randn(1, t, 2, d, generator=g) * 3).to(dtype)
    kx, vx = orc.stands_for(k), orc.stands_for(v)
    got = ops.kv4_attention(q.to(cuda), pool, z, table(starts, cuda))
    check_attention(got, q, kx, vx, starts, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("starts,t,h,group,d", [
    ([5000, 7], 1, 2, 1, 128),  # few rows over a long axis: split among CTAs
    ([20011], 1, 1, 1, 64),
    ([3000, 2999, 3100], 5, 1, 1, 64),
    ([2100], 1, 1, 8, 128),
    ([767, 768, 769], 1, 2, 1, 32),  # about the longest that is not split
    ([31 * i % 400 for i in range(70)], 1, 2, 1, 64),  # more requests than a warp's lanes
    ([1 + 97 * i % 2000 for i in range(40)], 1, 1, 2, 96),
    ([5, 0, 4000], 1, 16, 1, 32),
])
def test_attention_of_long_and_many_requests(cuda, dtype, starts, t, h, group, d):
    pool, slots, st, kx, vx = fill(cuda, dtype, starts, t, h, d, seed=d + t + 1)
    q = torch.randn(len(starts), t, h * group, d, generator=torch.Generator().manual_seed(d)).to(dtype)
    check_attention(ops.kv4_attention(q.to(cuda), pool, slots, st), q, kx, vx, starts, dtype)


@pytest.mark.parametrize("dtype", DTYPES[:2])
@pytest.mark.parametrize("starts,t,h,group,d", [
    ([6000, 200, 3000], 1, 4, 16, 64),  # shared heads of single tokens, several blocks a CTA
    ([2500, 131], 1, 2, 9, 128),
    ([4100], 5, 2, 4, 128),
    ([900, 0, 2500, 31], 20, 8, 1, 64),  # CTAs that end one segment and begin the next
    ([60 * i for i in range(10)], 130, 8, 4, 64),  # enough segments for one a CTA
    ([128], 257, 1, 1, 64),
    ([40, 333], 70, 2, 1, 32),  # one group of channels, three, and short ones
    ([1000], 3, 2, 5, 96),
    ([100, 0, 511], 50, 3, 2, 80),
    ([77], 140, 2, 1, 100),
    ([12, 260], 33, 1, 3, 7),
    ([5], 21, 2, 1, 33),
    ([0], 10, 1, 1, 1),
    ([300, 70], 40, 1, 1, 160),  # one block of operands and scores at a time
    ([128, 1000], 20, 2, 2, 192),
    ([63], 150, 1, 1, 224),
    ([1500, 2, 640], 130, 2, 1, 256),
    ([200], 4, 1, 3, 250),
])
def test_attention_on_the_tensor_cores(cuda, dtype, starts, t, h, group, d):
    assert on_tensor_cores(dtype, t, group)
    pool, slots, st, kx, vx = fill(cuda, dtype, starts, t, h, d, seed=d + t + 2)
    q = torch.randn(len(starts), t, h * group, d, generator=torch.Generator().manual_seed(d)).to(dtype)
    check_attention(ops.kv4_attention(q.to(cuda), pool, slots, st), q, kx, vx, starts, dtype)


@pytest.mark.parametrize("t,d", [(1, 128), (5, 96), (40, 128), (150, 64), (30, 256)])
@pytest.mark.parametrize("qp,kp,vp", [(60, -60, -80), (-70, 70, 100), (0, 0, 0)])
def test_bf16_magnitudes(cuda, t, d, qp, kp, vp):
    """bf16's range: queries, keys and values far from 1, tiles of different
    magnitudes, and tiles of zeros."""
    dtype, starts = torch.bfloat16, [333, 0]
    n = starts[0] + t
    k, v = rows(2, n, 2, d, dtype, seed=11, offset=False)
    tile = torch.arange(n) // 32
    k = (k.double() * 2.0 ** (kp - tile % 3)[None, :, None, None]).to(dtype)
    v = (v.double() * 2.0 ** (vp + tile % 7 - 3)[None, :, None, None]).to(dtype)
    k[:, 32:64], v[:, 64:96], k[:, -5:], v[:, -3:] = 0, 0, 0, 0
    q = (torch.randn(2, t, 2, d, generator=torch.Generator().manual_seed(t)).double() * 2.0 ** qp).to(dtype)
    pool = make_pool(cuda, 2, 2, n + 3, d, dtype)
    slots = table([1, 0], cuda)
    for i in range(2):
        m = starts[i] + t
        ops.kv4_append(k[i:i + 1, :m].to(cuda), v[i:i + 1, :m].to(cuda), pool, slots[i:i + 1], table([0], cuda))
    got = ops.kv4_attention(q.to(cuda), pool, slots, table(starts, cuda))
    check_attention(got, q, orc.stands_for(k), orc.stands_for(v), starts, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("t,group,d", [(1, 1, 128), (6, 1, 64), (40, 1, 128), (100, 2, 64), (3, 3, 80),
                                       (50, 1, 192)])
def test_nan_in_values_reaches_its_group_of_those_who_attend_it(cuda, dtype, t, group, d):
    """A value of NaN or infinity in one group's channels, a key of NaN further on:
    earlier rows' weights of zero undo both."""
    starts, h = [20, 300], 2
    n = max(starts) + t
    k, v = rows(2, n, h, d, dtype, seed=13)
    v[0, 20 + t // 2, 1, 33] = math.nan
    v[1, 300 + t // 3, 0, d - 1] = math.inf
    k[1, 300 + t - 1, 1, 2] = math.nan
    pool = make_pool(cuda, 2, h, n, d, dtype)
    slots = table([0, 1], cuda)
    for i in range(2):
        m = starts[i] + t
        ops.kv4_append(k[i:i + 1, :m].to(cuda), v[i:i + 1, :m].to(cuda), pool, slots[i:i + 1], table([0], cuda))
    q = torch.randn(2, t, h * group, d, generator=torch.Generator().manual_seed(t)).to(dtype)
    got = ops.kv4_attention(q.to(cuda), pool, slots, table(starts, cuda))
    kx, vx = orc.stands_for(k), orc.stands_for(v)
    want = orc.attention(q, kx, vx, starts)
    assert want.isnan().any() and not want.isnan().all()
    check_attention(got, q, kx, vx, starts, dtype)


def test_calls_at_once_on_two_streams_and_graphs(cuda):
    """Split requests on two streams at once, eager and captured: each call has its
    own workspace."""
    dtype, d = torch.bfloat16, 64
    streams = [torch.cuda.Stream() for _ in range(2)]
    calls, want = [], []
    for i, (starts, t, group) in enumerate([([4000, 9], 1, 1), ([1500], 4, 4)]):
        pool, slots, st, _, _ = fill(cuda, dtype, starts, t, 2, d, seed=20 + i)
        q = torch.randn(len(starts), t, 2 * group, d, generator=torch.Generator().manual_seed(i)).to(dtype).to(cuda)
        calls.append((q, pool, slots, st))
        want.append(ops.kv4_attention(*calls[-1]))
    torch.cuda.synchronize()
    graphs, outs = [], []
    for s, c in zip(streams, calls):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            outs.append(ops.kv4_attention(*c))
        graphs.append(g)
    got = [[], []]
    for _ in range(20):
        for i in (0, 1):
            with torch.cuda.stream(streams[i]):
                got[i].append(ops.kv4_attention(*calls[i]))
    torch.cuda.synchronize()
    for i in (0, 1):
        assert all(torch.equal(x, want[i]) for x in got[i])
    for _ in range(20):
        for i in (0, 1):
            outs[i].fill_(math.nan)
        torch.cuda.synchronize()
        for i in (0, 1):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        torch.cuda.synchronize()
        for i in (0, 1):
            assert torch.equal(outs[i], want[i])


def test_attention_of_strided_queries_into_out(cuda):
    """q as column views of a projection's output, aligned and not; out given."""
    dtype, starts, h = torch.bfloat16, [90, 20], 3
    for off, t, d in ((0, 1, 64), (8, 1, 64), (3, 1, 64), (0, 12, 64), (8, 12, 80), (3, 12, 128), (0, 9, 36)):
        pool, slots, st, kx, vx = fill(cuda, dtype, starts, t, h, d, seed=1)
        wide = torch.randn(2 * t, 3 * h * d + off, generator=torch.Generator().manual_seed(off)).to(dtype)
        q = wide[:, off:off + h * d].unflatten(1, (h, d)).unflatten(0, (2, t))
        qd = wide.to(cuda)[:, off:off + h * d].unflatten(1, (h, d)).unflatten(0, (2, t))
        memory = torch.full((2 * t * h * d + off,), math.nan, dtype=dtype, device=cuda)
        out = memory[off:].view(2, t, h * d)
        assert ops.kv4_attention(qd, pool, slots, st, out=out) is out
        check_attention(out, q, kx, vx, starts, dtype)
        assert memory[:off].isnan().all()


def test_a_row_that_reads_nan_reaches_only_those_who_attend_it(cuda):
    dtype, d = torch.bfloat16, 128
    k, v = rows(1, 40, 1, d, dtype, seed=2)
    k[0, 30, 0, 5] = math.nan
    pool = make_pool(cuda, 1, 1, 64, d, dtype)
    z = table([0], cuda)
    ops.kv4_append(k.to(cuda), v.to(cuda), pool, z, z)
    q = torch.randn(1, 1, 1, d, device=cuda).to(dtype)
    assert torch.isfinite(ops.kv4_attention(q, pool, z, table([29], cuda))).all()
    assert ops.kv4_attention(q, pool, z, table([30], cuda)).isnan().all()


@pytest.mark.parametrize("t", [1, 3, 40])
def test_bad_slots_and_positions_raise_the_error_word(cuda, t):
    dtype, h, d, max_seq = torch.bfloat16, 2, 64, 48
    pool = make_pool(cuda, 3, h, max_seq, d, dtype)
    good = rows(1, max_seq, h, d, dtype, seed=4)
    ops.kv4_append(good[0].to(cuda), good[1].to(cuda), pool, table([1], cuda), table([0], cuda))
    before = snapshot(pool)
    k, v = rows(1, t, h, d, dtype, seed=5)
    q = torch.randn(1, t, h, d).to(dtype).to(cuda)
    for slot, start in ((-1, 0), (3, 0), (1, -1), (1, max_seq), (1, 2 ** 31 - 1), (-2 ** 31, 0)):
        sl, st = table([slot], cuda), table([start], cuda)
        ops.kv4_append(k.to(cuda), v.to(cuda), pool, sl, st)
        assert _native.device_status() == RANGE
        for x, y in zip(before, snapshot(pool)):
            assert torch.equal(x, y)
        assert not ops.kv4_attention(q, pool, sl, st).any()
        assert _native.device_status() == RANGE
        kr, vr = ops.kv4_read(pool, sl, t, start_pos=st)
        assert not kr.any() and not vr.any()
        assert _native.device_status() == RANGE
    # a chunk that ends outside: the queries that fit are answered, the others are zeros
    kx, vx = orc.stands_for(good[0]), orc.stands_for(good[1])
    if t > 1:
        st = table([max_seq - 1], cuda)
        got = ops.kv4_attention(q, pool, table([1], cuda), st)
        assert _native.device_status() == RANGE
        check_attention(got[:, :1], q[:, :1].cpu(), kx, vx, [max_seq - 1], dtype, t)
        assert not got[:, 1:].any()


def test_the_same_slot_twice_keeps_the_first(cuda):
    dtype, h, d = torch.float16, 3, 64
    k, v = rows(4, 6, h, d, dtype, seed=6)
    pool = make_pool(cuda, 3, h, 32, d, dtype)
    # requests 0 and 2 overlap in slot 1; request 3 shares the slot but not the rows
    slots, starts = table([1, 0, 1, 1], cuda), table([4, 4, 9, 20], cuda)
    ops.kv4_append(k.to(cuda), v.to(cuda), pool, slots, starts)
    assert _native.device_status() == RANGE
    kr, _ = ops.kv4_read(pool, slots, 6, start_pos=starts)
    want = orc.stands_for(k).transpose(1, 2)
    for i in (0, 1, 3):
        check_values(kr[i], want[i], dtype)
    # reading and attending the same slot twice is fine
    q = torch.randn(2, 1, h, d).to(dtype).to(cuda)
    two = ops.kv4_attention(q[:1].expand(2, -1, -1, -1).contiguous(), pool, table([1, 1], cuda), table([9, 9], cuda))
    assert torch.equal(two[0], two[1]) or two.isnan().any()  # rows 0..3 were never written: NaN both times


def test_rows_beyond_four_gigabytes(cuda):
    """Codes at byte offsets past 32 bits (the pool's memory is mostly untouched)."""
    dtype, h, d, max_seq, slots = torch.bfloat16, 16, 128, 8192, 530
    pool = KV4Pool(slots=slots, heads=h, max_seq_len=max_seq, head_dim=d, device=cuda, dtype=dtype)
    assert pool.nbytes > 1 << 33
    n = 33
    k, v = rows(2, n, h, d, dtype, seed=8)
    sl = table([slots - 1, 7], cuda)
    z = table([0, 0], cuda)
    ops.kv4_append(k.to(cuda), v.to(cuda), pool, sl, z)
    kx, vx = orc.stands_for(k), orc.stands_for(v)
    check_values(ops.kv4_read(pool, sl, n)[0], kx.transpose(1, 2), dtype)
    q = torch.randn(2, 1, h, d).to(dtype)
    check_attention(ops.kv4_attention(q.to(cuda), pool, sl, table([n - 1] * 2, cuda)), q, kx, vx, [n - 1] * 2, dtype)


@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 128), (torch.float16, 64), (torch.float32, 80)])
def test_prefill_and_decode_together_in_a_captured_graph(cuda, dtype, d):
    """A prompt's rows appended and attended, then decode steps whose append and
    attention are captured once and replayed with moving positions."""
    b, h, t0, steps = 3, 2, 21, 6
    k, v = rows(b, t0 + steps, h, d, dtype, seed=9)
    kx, vx = orc.stands_for(k), orc.stands_for(v)
    q = torch.randn(b, t0 + steps, h, d, generator=torch.Generator().manual_seed(1)).to(dtype)
    pool = make_pool(cuda, 4, h, 64, d, dtype)
    slots, starts = table([2, 0, 3], cuda), table([0] * b, cuda)
    kd, vd, qd = k.to(cuda), v.to(cuda), q.to(cuda)
    ops.kv4_append(kd[:, :t0], vd[:, :t0], pool, slots, starts)
    got = ops.kv4_attention(qd[:, :t0], pool, slots, starts)
    check_attention(got, q[:, :t0], kx, vx, [0] * b, dtype)
    ks, vs, qs = (x[:, :1].clone() for x in (kd, vd, qd))
    starts.fill_(t0)
    ks.copy_(kd[:, t0:t0 + 1]), vs.copy_(vd[:, t0:t0 + 1])

    def step():
        ops.kv4_append(ks, vs, pool, slots, starts)
        return ops.kv4_attention(qs, pool, slots, starts)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(steps):
        ks.copy_(kd[:, t0 + i:t0 + i + 1]), vs.copy_(vd[:, t0 + i:t0 + i + 1]), qs.copy_(qd[:, t0 + i:t0 + i + 1])
        starts.fill_(t0 + i)
        graph.replay()
        check_attention(out, q[:, t0 + i:t0 + i + 1], kx, vx, [t0 + i] * b, dtype)


def test_results_repeat_bit_for_bit(cuda):
    dtype, starts = torch.bfloat16, [900, 33, 512]
    for t in (1, 4, 140):
        pool, slots, st, _, _ = fill(cuda, dtype, starts, t, 2, 128, seed=t)
        q = torch.randn(3, t, 4, 128, device=cuda).to(dtype)
        first = ops.kv4_attention(q, pool, slots, st)
        for _ in range(3):
            assert torch.equal(first, ops.kv4_attention(q, pool, slots, st))


# ------------------------------------------------------------- in the decoder
def small_engine(**kw):
    cfg = DecoderConfig(**{**dict(vocab_size=64, hidden_size=128, num_heads=2, num_layers=2, intermediate_size=256,
                                  max_seq_len=96, seed=17), **kw.pop("cfg", {})})
    return cfg, Engine(cfg, context=ParallelContext.from_env(device="cuda"), max_requests=4, init=kw.pop("init", "reference"),
                       **kw)


def decoder_reference(cfg, tokens, dtype):
    """Logits [B, T, V] in float64 of the reference decoder's weights (rounded
    to dtype) with every layer's keys and values quantised as they are written."""
    ref = TinyDecoder(cfg).to(dtype).double()
    x = ref.token_embedding(tokens) + ref.position_embedding(torch.arange(tokens.shape[1]))
    b, t, h = x.shape
    for blk in ref.blocks:
        y = blk.ln1(x)
        q, k, v = (f(y).view(b, t, cfg.num_heads, cfg.head_dim) for f in (blk.q, blk.k, blk.v))
        kx, vx = (orc.stands_for(z.detach().to(dtype)) for z in (k, v))
        x = x + blk.o(orc.attention(q, kx, vx, [0] * b))
        x = x + blk.down(torch.nn.functional.gelu(blk.up(blk.ln2(x)), approximate="tanh"))
    return ref.lm_head(ref.final_norm(x)).detach()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("ln", ["fold", "prologue", "kernel"])
def test_engine_with_a_4_bit_cache(cuda, dtype, ln):
    """Prefill, captured decode steps and per-request positions through the
    engine, against the decoder whose keys and values are quantised in float64.

    A step is at most 2^-4 of a group's span wide (15 steps, half a step either
    side); a rounding elsewhere in the decoder moves a number across a border
    now and then and so by one step.  The logits are therefore compared at 2e-2
    of their scale for 16 bits, as the decoder's own tests are, and at 2e-3 for
    fp32."""
    cfg, eng = small_engine(dtype=dtype, kv_bits=4)
    eng.decoder.decode_ln = ln
    assert eng.decoder.cache.k_pool == {} and len(eng.decoder.cache.kv4_pool) == 2
    tokens = torch.randint(0, 64, (3, 60), generator=torch.Generator().manual_seed(2))
    want = decoder_reference(cfg, tokens, dtype)
    rel = 2e-3 if dtype == torch.float32 else 2e-2
    atol = rel * float(want.abs().max())
    got = [eng.forward(tokens[:, :55], (5, 6, 7), 0)]
    got += [eng.forward(tokens[:, i:i + 1], (5, 6, 7), i) for i in range(55, 60)]
    torch.testing.assert_close(torch.cat([g.cpu() for g in got], 1).double(), want, rtol=0, atol=atol)
    eng.close()


def test_generate_with_a_4_bit_cache_eager_and_captured(cuda):
    outs = []
    for graphs in (True, False):
        _, eng = small_engine(dtype=torch.bfloat16, kv_bits=4)
        eng.decoder.use_cuda_graphs = graphs
        outs.append((eng.generate([[1, 2, 3, 4, 5], [6, 7, 8, 9, 10]], 20),
                     eng.generate_mixed([[1, 2, 3], [4, 5, 6, 7, 8, 9, 10], [11]], 12)))
        eng.close()
    assert outs[0] == outs[1]


def test_cache_append_returns_the_prefixes_it_stands_for(cuda):
    for dtype in DTYPES:
        c = KVCache(layer_ids=(3, 4), num_heads=2, head_dim=48, max_seq_len=20, max_requests=3, device=cuda,
                    dtype=dtype, kv_bits=4)
        c.reserve((10, 11))
        k, v = rows(2, 9, 2, 48, dtype, seed=12)
        for lo, hi in ((0, 5), (5, 6), (6, 9)):
            for lid in (3, 4):
                pk, pv = c.append(lid, (10, 11), k[:, lo:hi].transpose(1, 2).to(cuda),
                                  v[:, lo:hi].transpose(1, 2).to(cuda), lo)
                check_values(pk, orc.stands_for(k[:, :hi]).transpose(1, 2), dtype)
                check_values(pv, orc.stands_for(v[:, :hi]).transpose(1, 2), dtype)
        with pytest.raises(CacheError):
            c.append(5, (10,), k[:1, :1].transpose(1, 2).to(cuda), v[:1, :1].transpose(1, 2).to(cuda), 9)
