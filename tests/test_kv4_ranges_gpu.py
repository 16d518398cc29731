"""The 4-bit key/value cache where numbers of very different sizes meet: a row's
result depends on the positions that it attends, each by its weight, and on
nothing else.  Bounds are taken over the attended rows only (``attended_bound``);
the definition is oracle/kv4.py in float64."""

import math

import pytest
import torch

from forgeml_b200 import _native
from forgeml_b200.nebula import KV4Pool, ops
from oracle import kv4 as orc

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
LEVELS = {torch.bfloat16: 65530, torch.float16: 8388600, torch.float32: 8388600}


@pytest.fixture(autouse=True)
def clean_status(cuda):
    _native.device_status()
    yield
    assert _native.device_status() == 0


def table(values, cuda):
    return torch.tensor(values, dtype=torch.int32, device=cuda)


def filled(cuda, k, v, slots=1):
    """A pool whose slot 0 holds k and v [1, n, H, D], and those rows in float64."""
    _, n, h, d = k.shape
    pool = KV4Pool(slots=slots, heads=h, max_seq_len=n, head_dim=d, device=cuda, dtype=k.dtype)
    pool.data.fill_(255)
    ops.kv4_append(k.to(cuda), v.to(cuda), pool, table([0], cuda), table([0], cuda))
    return pool, orc.stands_for(k), orc.stands_for(v)


def attended_bound(q, kx, vx, starts, dtype, tc, terms=None):
    """float64 [B, T, QH * D]: what a kernel may be off by before the output's
    rounding, from the rows that a query attends.  e = 2^-24, w the weights, A =
    sum w |v| of an output, n the attended positions.  Weights whose scores are off
    by x are off by expm1(x) of themselves against their sum.

    Up to 8 rows of a head, or fp32 (a group of 32 channels is z + c s, its span
    15 s; a = |z| + 15 s, for fp32 |z + 8 s| + 8 s):
      scores    q as an integer q / max|q| * 1.2e8, rounded to fp32, then to the
                integer; put together in fp32, (G + 8) e of scale * sum |q| a (in
                float64 for fp32).  The exponent: e times the distance from the
                maximum.
      weights   exponential 2^-22, and once more each time that the maximum moves.
      digits    w s goes as an integer of units of at most 1.25 max (w s) / levels,
                and what a lane rounds off is carried to its next position: the
                rounding of a position is off by r_j = e_(j-1) - e_j, |e| at most one
                unit, and sum r_j c_j = sum e_j (c_(j+1) - c_j) is at most a unit times
                15 for each of the ``terms`` positions where the lane's next code is
                another (n of them unless the caller knows better).
      sums      4 (n / 32 + 40) e of sum w a.
    On the tensor cores, u = 2^-11 the rounding to fp16.  bf16's operands are scaled
    by powers of two to 2^12 at least for the largest number of a position or, where
    32 neighbouring positions differ by less than 2^10, of those; the largest weight
    times value of a row to 2^13 at least, or 2^3 where neighbours differ; M the
    largest |number| of a position.
      scores    u of every |q k|, the products' sums (d + 8) 2^-23, and the subnormal
                step: 2^-25 (fp16), 2^-37 of the largest |q|, 2^-26 of M for the keys;
                the exponent as above.
      weights   2^-22 each and per move; weights and values rounded, 2 u A; the
                subnormal steps: of a value 2^-25 (fp16) or 2^-26 M, of a weight 2^-26
                of the row's largest w M; sums (n / 16 + 40) 2^-23 A."""
    b, t, qh, d = q.shape
    q = q.detach().cpu().double()
    h, u, e = kx.shape[2], 2.0 ** -11, 2.0 ** -24
    group, scale, wide = qh // h, 1 / math.sqrt(d), dtype == torch.float32
    bound = torch.empty(b, t, qh, d, dtype=torch.float64)

    def spans(x, wide):
        a, st = torch.empty_like(x), torch.empty_like(x)
        for c0 in range(0, d, 32):
            g = x[..., c0:c0 + 32]
            z, s15 = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True) - g.amin(-1, keepdim=True)
            a[..., c0:c0 + 32] = ((z + s15 * 8 / 15).abs() + s15 * 8 / 15) if wide else z.abs() + s15
            st[..., c0:c0 + 32] = s15 / 15
        return a, st

    ka, _ = spans(kx, False)
    va, vs = spans(vx, wide)
    for i in range(b):
        for j in range(t):
            n = int(starts[i]) + j + 1
            moves = n / 32 + 1
            for hq in range(qh):
                hk = hq // group
                kh, vh, qi = kx[i, :n, hk], vx[i, :n, hk], q[i, j, hq]
                sc = kh @ qi * scale
                w = torch.softmax(sc, 0)
                A = w @ vh.abs()
                far = sc.max() - sc
                if tc:
                    km, vm = kh.abs().amax(1), vh.abs().amax(1)
                    x = (u + (d + 8) * 2 * e) * (kh.abs() @ qi.abs()) * scale + 2 * e * (far + sc.abs())
                    if dtype == torch.float16:
                        x = x + 2.0 ** -25 * (qi.abs().sum() + kh.abs().sum(1)) * scale
                        step = 2.0 ** -25
                    else:
                        x = x + (2.0 ** -26 * qi.abs().sum() * km + 2.0 ** -37 * qi.abs().max() * kh.abs().sum(1)) * scale
                        step = 2.0 ** -26 * (w @ vm)
                    rel = moves / 4 * 2.0 ** -22 + 2.0 ** -22 + x
                    other = 2 * u * A + step + n * 2.0 ** -26 * (w * vm).max() + (n / 16 + 40) * 2 * e * A
                else:
                    small = ka[i, :n, hk] @ qi.abs() * scale
                    x = e * small + 0.6 / 1.2e8 * qi.abs().max() * scale * ka[i, :n, hk].sum(1) + e * far
                    x = x + (0 if wide else (-(-d // 32) + 8) * e * small)
                    rel = x + moves * 2.0 ** -22
                    unit = 1.25 * (w[:, None] * vs[i, :n, hk]).amax(0) / LEVELS[dtype]
                    other = 15 * unit * (n if terms is None else min(n, terms)) + 4 * (n / 32 + 40) * e * (w @ va[i, :n, hk])
                off = w * torch.expm1(rel)
                bound[i, j, hq] = off @ vh.abs() + off.sum() * A + other
    return bound.reshape(b, t, qh * d)


def check(got, q, kx, vx, starts, dtype, tc, terms=None, rows=None):
    """rows: how many of the call's query rows are looked at (all)."""
    b = q.shape[0]
    kx, vx = (x.expand(b, -1, -1, -1) for x in (kx, vx))
    rows = q.shape[1] if rows is None else rows
    q, got = q[:, :rows], got[:, :rows].cpu().double()
    n = max(starts) + rows
    want = orc.attention(q, kx[:, :n], vx[:, :n], starts)
    f = torch.finfo(dtype)
    tol = attended_bound(q, kx[:, :n], vx[:, :n], starts, dtype, tc, terms) * (1 + f.eps)
    tol = tol + f.eps / 2 * want.abs() + f.tiny * f.eps / 2
    assert want.isfinite().all() and tol.isfinite().all()
    err = (got - want).abs()
    assert (err <= tol).all(), (float(err.max()), float((err / tol).max()), float(want.abs().max()))


def gen(seed):
    return torch.Generator().manual_seed(seed)


MANY = 128  # requests of 16 heads, all reading the same slot: more segments than the chip has warps


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("power", [7, 10, 14, 26])
def test_a_large_value_of_vanishing_weight_among_later_rows(cuda, dtype, power):
    """Position 5's value is 2^power times the others', the first 32 positions score
    far below the later ones.  One warp holds whole segments of 1024 positions."""
    n, h, d = 1024, 16, 32
    if dtype == torch.float16:
        power = min(power, 12)
    dirn = torch.where(torch.rand(h, d, generator=gen(1)) < 0.5, -1.0, 1.0)
    k = 0.3 * torch.randn(1, n, h, d, generator=gen(2))
    gap = 10 + power  # nats
    k[:, :32] -= gap / math.sqrt(d) * dirn
    v = torch.randn(1, n, h, d, generator=gen(3))
    v[:, 5] *= 2.0 ** power
    k, v = k.to(dtype), v.to(dtype)
    q = (dirn + 0.1 * torch.randn(MANY, 1, h, d, generator=gen(4))).to(dtype)
    pool, kx, vx = filled(cuda, k, v)
    got = ops.kv4_attention(q.to(cuda), pool, table([0] * MANY, cuda), table([n - 1] * MANY, cuda))
    check(got[:2], q[:2], kx, vx, [n - 1] * 2, dtype, False)
    check(got[-2:], q[-2:], kx, vx, [n - 1] * 2, dtype, False)


@pytest.mark.parametrize("dtype", DTYPES)
def test_many_small_weights_beside_a_large_one(cuda, dtype):
    """One position takes nearly all the weight, with channels of zero; each of the
    8191 others has a weight of a fraction of the integers' unit.  Together they are
    what those channels hold."""
    n, h, d = 8192, 16, 32
    dirn = torch.where(torch.rand(h, d, generator=gen(1)) < 0.5, -1.0, 1.0)
    small = 0.3 * 1.25 / LEVELS[dtype]
    half = -math.log(small) / 2 / math.sqrt(d)
    k = (-half * dirn).expand(1, n, h, d).clone()
    k[:, 0] = half * dirn
    v = torch.randn(h, d, generator=gen(3)).abs().expand(1, n, h, d).clone()
    v[:, 0] = torch.arange(d) % 2 * v[:, 1].amax(-1, keepdim=True)
    k, v = k.to(dtype), v.to(dtype)
    q = dirn.expand(MANY, 1, h, d).to(dtype)
    pool, kx, vx = filled(cuda, k, v)
    got = ops.kv4_attention(q.to(cuda), pool, table([0] * MANY, cuda), table([n - 1] * MANY, cuda))
    # the codes differ behind the first position and at the ends of 32 lanes in at most 4 shares
    for i in (0, 77, MANY - 1):
        check(got[i:i + 1], q[i:i + 1], kx, vx, [n - 1], dtype, False, terms=2 + 4 * 32)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("exponent", [-80, -100, -110, -118])
def test_values_near_the_smallest_numbers(cuda, dtype, exponent):
    n, h, d = 1024, 16, 32
    k = torch.randn(1, n, h, d, generator=gen(2)).to(dtype)
    v = (torch.randn(1, n, h, d, generator=gen(3)) * 2.0 ** exponent).to(dtype)
    q = torch.randn(MANY, 1, h, d, generator=gen(4)).to(dtype)
    pool, kx, vx = filled(cuda, k, v)
    got = ops.kv4_attention(q.to(cuda), pool, table([0] * MANY, cuda), table([n - 1] * MANY, cuda))
    check(got[:2], q[:2], kx, vx, [n - 1] * 2, dtype, False)


@pytest.mark.parametrize("lead", [0.0, 2.0 ** -30])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_steps_that_grow_by_many_powers_of_two(cuda, dtype, lead):
    """Constant or tiny values first, then larger and larger ones, then tiny again."""
    n, h, d = 1024, 16, 32
    k = 0.3 * torch.randn(1, n, h, d, generator=gen(2)).to(dtype)
    v = torch.randn(1, n, h, d, generator=gen(3))
    v[:, :100] *= lead
    for i, x in enumerate((-118, -60, 0, 40, 100)):
        v[:, 100 + 64 * i:164 + 64 * i] *= 2.0 ** x
    v[:, 420:] *= 2.0 ** -100
    v = v.to(dtype)
    q = torch.randn(MANY, 1, h, d, generator=gen(4)).to(dtype)
    pool, kx, vx = filled(cuda, k, v)
    for last in (90, 150, 230, 300, n - 1):
        got = ops.kv4_attention(q.to(cuda), pool, table([0] * MANY, cuda), table([last] * MANY, cuda))
        check(got[:1], q[:1], kx, vx, [last], dtype, False)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("qp,kp", [(-88, 90), (-20, 100), (60, -64)])
def test_scores_of_large_keys_and_small_queries(cuda, dtype, qp, kp):
    n, h, d = 200, 4, 64
    k = (torch.randn(1, n, h, d, generator=gen(2)) * 2.0 ** kp).to(dtype)
    if qp + kp > 8:
        # such scores leave one position; it is apart from the others by far
        k[0, :, :, :] = k[0, :, :, :].float().mul(2.0 ** -40).to(dtype)
        k[0, 77] = k[0, 77].float().mul(2.0 ** 40).to(dtype)
    v = torch.randn(1, n, h, d, generator=gen(3)).to(dtype)
    q = (torch.randn(1, 1, h, d, generator=gen(4)) * 2.0 ** qp).to(dtype)
    if qp + kp > 8:  # towards that position
        q = (k[:, 77:78].float().sign() * q.float().abs()).to(dtype)
    pool, kx, vx = filled(cuda, k, v)
    got = ops.kv4_attention(q.to(cuda), pool, table([0], cuda), table([n - 1], cuda))
    if qp + kp > 8:
        want = vx[0, 77].reshape(-1)
        f = torch.finfo(dtype)
        err = (got[0, 0].cpu().double() - want).abs()
        assert (err <= f.eps / 2 * want.abs() + 200 * 2.0 ** -24 * want.abs().max() + 32 * 20 / LEVELS[dtype]).all(), err.max()
    else:
        check(got, q, kx, vx, [n - 1], dtype, False)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("power", [7, 14, 18, 22, 26, 40, 100])
@pytest.mark.parametrize("at,d", [(110, 64), (110, 128), (64, 160), (10, 64)])
def test_a_prompt_row_does_not_depend_on_a_large_later_value(cuda, dtype, power, at, d):
    """Position ``at``'s value is 2^power times the others'."""
    t, h = 128, 2
    if dtype == torch.float16:
        power = min(power, 13)
    k, v = (torch.randn(1, t, h, d, generator=gen(s)) for s in (2, 3))
    v[:, at] *= 2.0 ** power
    k, v = k.to(dtype), v.to(dtype)
    q = torch.randn(1, t, h, d, generator=gen(4)).to(dtype)
    pool, kx, vx = filled(cuda, k, v)
    got = ops.kv4_attention(q.to(cuda), pool, table([0], cuda), table([0], cuda))
    check(got, q, kx, vx, [0], dtype, True)


@pytest.mark.parametrize("power", [14, 26, 30, 40, 100])
@pytest.mark.parametrize("at,d", [(110, 64), (110, 192), (64, 64)])
def test_a_prompt_row_does_not_depend_on_a_large_later_key(cuda, power, at, d):
    dtype, t, h = torch.bfloat16, 128, 2
    k, v = (torch.randn(1, t, h, d, generator=gen(s)) for s in (2, 3))
    k[:, at] *= 2.0 ** power
    k, v = k.to(dtype), v.to(dtype)
    q = torch.randn(1, t, h, d, generator=gen(4)).to(dtype)
    pool, kx, vx = filled(cuda, k, v)
    got = ops.kv4_attention(q.to(cuda), pool, table([0], cuda), table([0], cuda))
    check(got, q, kx, vx, [0], dtype, True, rows=at)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("power", [7, 14, 18, 22, 26, 60])
@pytest.mark.parametrize("at", [5, 40, 200])
def test_a_large_value_of_vanishing_weight_in_a_prompt(cuda, dtype, power, at):
    """Scores of the rows around ``at`` lie far below the others'."""
    t, h, d, start = 40, 2, 64, 300
    if dtype == torch.float16:
        power = min(power, 13)
    dirn = torch.where(torch.rand(h, d, generator=gen(1)) < 0.5, -1.0, 1.0)
    k = 0.3 * torch.randn(1, start + t, h, d, generator=gen(2))
    k[:, at // 32 * 32:at // 32 * 32 + 32] -= (10 + power) / math.sqrt(d) * dirn
    v = torch.randn(1, start + t, h, d, generator=gen(3))
    v[:, at] *= 2.0 ** power
    k, v = k.to(dtype), v.to(dtype)
    q = (dirn + 0.1 * torch.randn(1, t, h, d, generator=gen(4))).to(dtype)
    pool, kx, vx = filled(cuda, k, v)
    got = ops.kv4_attention(q.to(cuda), pool, table([0], cuda), table([start], cuda))
    check(got, q, kx, vx, [start], dtype, True)


@pytest.mark.parametrize("dtype,size", [(torch.float16, 3e4), (torch.bfloat16, 3e4), (torch.bfloat16, 1e12), (torch.float32, 1e12)])
@pytest.mark.parametrize("t,d", [(1, 64), (9, 64), (9, 192)])
def test_scores_beyond_what_their_maximum_keeps(cuda, dtype, size, t, d):
    """One position is ahead of the others by far; its weight is 1 whatever fp32 keeps of
    the scores."""
    n, h = 200, 2
    dirn = torch.where(torch.rand(h, d, generator=gen(1)) < 0.5, -1.0, 1.0)
    k = torch.randn(1, n, h, d, generator=gen(2))
    k[:, 77] = size * dirn
    k, v = k.to(dtype), torch.randn(1, n, h, d, generator=gen(3)).to(dtype)
    q = (size * (dirn + 0.1 * torch.randn(1, t, h, d, generator=gen(4)))).to(dtype)
    pool, kx, vx = filled(cuda, k, v)
    got = ops.kv4_attention(q.to(cuda), pool, table([0], cuda), table([n - t], cuda)).cpu().double()
    want = vx[0, 77].reshape(-1)
    # the value and the output rounded; p s as an integer, 15 codes; fp32 sums of z and c s
    u = max(torch.finfo(dtype).eps / 2, 2.0 ** -11 if t > 8 and dtype != torch.float32 else 0)
    off = 2 * u * want.abs() + (20 / LEVELS[dtype] + 40 * 2.0 ** -24) * want.abs().max()
    assert ((got[0] - want).abs() <= off).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_many_small_weights_beside_a_large_one_on_the_tensor_cores(cuda, dtype):
    """As above, with weights below half of fp16's smallest step."""
    n, h, d, t, b = 8192, 16, 32, 9, 20
    dirn = torch.where(torch.rand(h, d, generator=gen(1)) < 0.5, -1.0, 1.0)
    half = 25.5 * math.log(2) / 2 / math.sqrt(d)
    k = (-half * dirn).expand(1, n, h, d).clone()
    k[:, 0] = half * dirn
    v = torch.randn(h, d, generator=gen(3)).abs().expand(1, n, h, d).clone()
    v[:, 0] = torch.arange(d) % 2 * v[:, 1].amax(-1, keepdim=True)
    k, v = k.to(dtype), v.to(dtype)
    q = dirn.expand(b, t, h, d).to(dtype)
    pool, kx, vx = filled(cuda, k, v)
    got = ops.kv4_attention(q.to(cuda), pool, table([0] * b, cuda), table([n - t] * b, cuda))
    check(got[:1], q[:1], kx, vx, [n - t], dtype, True, rows=2)


def borders(dtype):
    """Groups [n, 32] whose numbers lie beside a border k + 1/2 by less than fp32 keeps
    of x - min."""
    far = {torch.bfloat16: 2.0 ** -40, torch.float16: 2.0 ** -23, torch.float32: 2.0 ** -40}[dtype]
    groups = []
    for sign in (1, -1):
        g = torch.zeros(32, dtype=torch.float64)
        g[0], g[1] = -7.5, 7.5  # step 1: 0 is a border
        g[2], g[3], g[4] = sign * far, 0.5, -1.0
        groups.append(g)
        g = torch.arange(32).double() % 16 + 0.5  # step 1 from a minimum beside 0
        g[0], g[1] = sign * far, 15.0
        g[15] = 1.0
        g = g.clamp(max=15.0)
        g[16] = sign * far
        groups.append(torch.where(g < 0, sign * far, g))
        groups.append(g * 64)
        groups.append(g.flip(0) / 8)
    return torch.stack(groups).to(dtype)


@pytest.mark.parametrize("dtype", DTYPES)
def test_numbers_beside_a_border_by_less_than_fp32_keeps(cuda, dtype):
    x = borders(dtype)
    n = x.shape[0]
    more = torch.randn(64, 32, generator=gen(1)).to(dtype)
    more[:, ::3] *= torch.tensor(2.0 ** -12).to(dtype)
    x = torch.cat([x, more]).view(1, n + 64, 1, 32)
    k = torch.cat([x, x.roll(1, 1)], -1)  # two groups a row
    pool = KV4Pool(slots=1, heads=1, max_seq_len=n + 64, head_dim=64, device=cuda, dtype=dtype)
    zero = table([0], cuda)
    ops.kv4_append(k.to(cuda), k.flip(-1).to(cuda), pool, zero, zero)
    f = torch.finfo(dtype)
    for got, src in zip(ops.kv4_read(pool, zero, n + 64), (k, k.flip(-1))):
        want = orc.stands_for(src).transpose(1, 2)
        got = got.cpu().double()
        assert ((got - want).abs() <= (f.eps / 2 + 2.0 ** -24) * want.abs() + f.tiny * f.eps / 2).all()


def test_reading_and_attending_a_slot_twice_in_a_batch(cuda):
    """Every row written, so that the numbers are compared."""
    dtype, h, d, n = torch.float16, 3, 64, 40
    k, v = (torch.randn(1, n, h, d, generator=gen(s)).to(dtype) for s in (1, 2))
    pool, kx, vx = filled(cuda, k, v, slots=2)
    for t in (1, 12):
        q = torch.randn(1, t, h, d, generator=gen(3)).to(dtype)
        got = ops.kv4_attention(q.expand(2, -1, -1, -1).contiguous().to(cuda), pool, table([0, 0], cuda),
                                table([n - t] * 2, cuda))
        for i in range(2):
            check(got[i:i + 1], q, kx, vx, [n - t], dtype, t > 8)
    kr, vr = ops.kv4_read(pool, table([0, 0], cuda), n)
    assert torch.equal(kr[0], kr[1]) and torch.equal(vr[0], vr[1])
