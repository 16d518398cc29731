"""Measured cases of the 4-bit key/value cache: quantising rows as they are
written, reading them back, and attention over the cache.

Format.  A row is one position of one key/value head: ``head_dim`` numbers of
type T.  Its channels form groups of 32 (the last may be shorter).  A group
with minimum ``z`` and maximum ``h`` keeps ``z``, the step
``s = T((h - z) / 15)`` and, for each number x, the code
``c = round((x - z) / s)``, ties to even, limited to 0..15 (0 where s is 0).
It stands for ``z + c * s``.

Operators.
  append     k, v [B, T, H, D] become rows start..start+T-1 of each request's
             slot; the rows just written are read back [B, H, T, D].
  read       rows 0..count-1 of each request's slot, [B, H, count, D].
  attention  query t of request b sits at position start[b] + t and attends
             the rows 0..start[b]+t of the request's slot; query head h reads
             key/value head h // group.  [B, T, H * group * D].
"""

import math

import torch

own = False

GROUP = 32
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZES = {"bf16": 2, "fp16": 2, "fp32": 4}


# ------------------------------------------------------------------ the cases
def listed():
    def case(name, op, dtype, batch, t, heads, dim, lo, hi, max_seq, group=1):
        return {"name": name, "op": op, "dtype": dtype, "batch": batch, "t": t, "heads": heads, "group": group,
                "dim": dim, "lo": lo, "hi": hi, "max_seq": max_seq}

    return [
        # a decode step's new rows: 32 requests, 16 heads of 128, all at their own position
        case("append-step", "append", "bf16", 32, 1, 16, 128, 512, 639, 2048),
        # a prefill's rows: 32 prompts of 512 tokens
        case("append-prompts", "append", "bf16", 32, 512, 16, 128, 0, 0, 2048),
        # a chunk that starts inside a half-full slot, full precision, a head size that ends inside a group
        case("append-odd", "append", "fp32", 3, 333, 5, 80, 10, 77, 1000),
        # a cohort's prefix handed on in its own type (one pipeline stage's heads of 64)
        case("read-prefix", "read", "fp16", 8, 1000, 12, 64, 0, 0, 2048),
        # every slot of a full pool: 32 requests of 2048 positions, 16 heads of 128
        case("read-full", "read", "bf16", 32, 2048, 16, 128, 0, 0, 2048),
        # one short request: the latency of a single token
        case("attend-one", "attention", "bf16", 1, 1, 16, 128, 130, 130, 2048),
        # the decode step of 32 requests that generate 128 tokens after 512
        case("attend-step", "attention", "bf16", 32, 1, 16, 128, 512, 639, 2048),
        # 64 requests of mixed prompt lengths on one of four tensor-parallel ranks
        case("attend-mixed", "attention", "bf16", 64, 1, 8, 128, 128, 2303, 4096),
        # few rows over a long axis
        case("attend-long", "attention", "bf16", 1, 1, 16, 128, 100001, 100001, 131072),
        # query heads that share key/value heads
        case("attend-shared", "attention", "fp16", 16, 1, 8, 128, 4000, 8190, 8192, 4),
        # a few drafted tokens checked at once, full precision
        case("attend-draft", "attention", "fp32", 6, 5, 12, 64, 700, 1501, 2048),
        # prompts: every token of a chunk attends what came before it
        case("attend-prompts", "attention", "bf16", 8, 1000, 16, 128, 0, 1048, 2048),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        op = rng.choice(("append", "read", "attention", "attention", "attention"))
        dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
        dim = rng.choice((32, 64, 64, 80, 96, 128, 128, 128, 192, 256))
        heads = _spread(rng, 1, 32)
        batch = _spread(rng, 1, 64)
        group = 1
        lo = hi = 0
        if op == "append":
            t = rng.choice((1, _spread(rng, 2, 2048)))
            lo = rng.randrange(0, 500)
            hi = lo + rng.randrange(0, 1500)
        elif op == "read":
            t = _spread(rng, 1, 4096)
        else:
            group = rng.choice((1, 1, 1, 2, 4, 7, 8))
            t = rng.choice((1, 1, 1, _spread(rng, 2, 16), _spread(rng, 17, 1500)))
            hi = _spread(rng, 1, 60000)
            lo = rng.randrange(0, hi + 1)
        max_seq = hi + t + rng.randrange(0, 300)
        c = {"op": op, "dtype": dtype, "batch": batch, "t": t, "heads": heads, "group": group, "dim": dim,
             "lo": lo, "hi": hi, "max_seq": max_seq}
        w = work(c)
        if batch * heads * max_seq * dim <= 1 << 28 and w["flops"] <= 6.7e10 and w["bytes"] <= 7.0e8:
            # the plain form keeps the scores in 32 bits
            if op != "attention" or batch * heads * group * t * (hi + t) <= 1 << 29:
                return c


def _starts(case):
    """Each request's first position: spread evenly over lo..hi, not in order."""
    b, lo, hi = case["batch"], case["lo"], case["hi"]
    if b == 1:
        return [hi]
    return [lo + (hi - lo) * ((i * 7 + 3) % b) // (b - 1) for i in range(b)]


def work(case):
    b, t, h, d, e = case["batch"], case["t"], case["heads"], case["dim"], SIZES[case["dtype"]]
    groups = -(-d // GROUP)
    row = 2 * h * (-(-d // 2) + 2 * groups * e)  # a position's keys and values, all heads
    if case["op"] == "append":
        # the rows in, the quantised rows out and in again, the values out
        return {"bytes": b * t * (4 * h * d * e + 2 * row), "flops": 8 * b * t * 2 * h * d}
    if case["op"] == "read":
        return {"bytes": b * t * (row + 2 * h * d * e), "flops": 2 * b * t * 2 * h * d}
    starts = _starts(case)
    keys = sum(s + t for s in starts)
    pairs = sum(t * s + t * (t + 1) // 2 for s in starts)
    qh = h * case["group"]
    return {"bytes": keys * row + 2 * b * t * qh * d * e, "flops": 4 * pairs * qh * d}


# ------------------------------------------------------------------ the state
def _rows(g, batch, n, heads, dim, dtype):
    """Keys and values as a decoder's projections give them, [B, n, H, D]:
    keys with some channels far from zero, values around zero."""
    dev = torch.device("cuda")
    k = torch.randn(batch, n, heads, dim, device=dev, dtype=dtype, generator=g)
    v = torch.randn(batch, n, heads, dim, device=dev, dtype=dtype, generator=g)
    centre = torch.randn(heads, dim, device=dev, generator=g)
    centre = centre + 4.0 * centre.sign() * (torch.rand(heads, dim, device=dev, generator=g) > 0.94)
    k += centre.to(dtype)
    return k, v


def prepare(case, seed):
    dtype = DTYPES[case["dtype"]]
    b, t, h, d = case["batch"], case["t"], case["heads"], case["dim"]
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    slots = b + 2
    slot_of = torch.randperm(slots, generator=g, device=dev)[:b].to(torch.int32)
    starts = torch.tensor(_starts(case), dtype=torch.int32).to(dev)
    st = {"case": case, "slot_of": slot_of, "starts": starts}
    if case["op"] == "append":
        st["k"], st["v"] = _rows(g, b, t, h, d, dtype)
        held = None
    else:
        n = t if case["op"] == "read" else max(_starts(case)) + t
        held = _rows(g, b, n, h, d, dtype)
        if case["op"] == "attention":
            st["q"] = torch.randn(b, t, h * case["group"], d, device=dev, dtype=dtype, generator=g)
    if own:
        from forgeml_b200.nebula import KV4Pool, ops

        st["pool"] = KV4Pool(slots=slots, heads=h, max_seq_len=case["max_seq"], head_dim=d, device=dev, dtype=dtype)
        if held is not None:
            ops.kv4_append(held[0], held[1], st["pool"], slot_of, torch.zeros_like(starts))
    elif held is not None:
        st["held"] = tuple(_quantise(x.transpose(1, 2)) for x in held)
    return st


# ------------------------------------------------------------ the plain forms
def _grouped(x):
    """[..., D] as [..., groups, 32]; a short last group repeats its last channel."""
    d = x.shape[-1]
    pad = -d % GROUP
    if pad:
        x = torch.cat([x, x[..., -1:].expand(*x.shape[:-1], pad)], dim=-1)
    return x.reshape(*x.shape[:-1], -1, GROUP)


def _quantise(x):
    """codes [..., groups, 32] (uint8), step and minimum [..., groups, 1] in x's
    type, and D.  Quotients next to a border need the 64 bits."""
    x = x.contiguous()
    codes, steps, lows = [], [], []
    for part in x.split(max(1, (1 << 25) // max(1, x[0].numel()))):
        gr = _grouped(part)
        low, high = gr.amin(-1, keepdim=True), gr.amax(-1, keepdim=True)
        step = ((high.double() - low.double()) / 15).to(x.dtype)
        c = torch.round((gr.double() - low.double()) / step.double()).clamp(0, 15)
        codes.append(torch.where(step > 0, c, torch.zeros_like(c)).to(torch.uint8))
        steps.append(step)
        lows.append(low)
    return torch.cat(codes), torch.cat(steps), torch.cat(lows), x.shape[-1]


def _values(quantised):
    codes, step, low, d = quantised
    x = codes.float() * step.float() + low.float()
    return x.reshape(*x.shape[:-2], -1)[..., :d]


def _plain(state):
    case = state["case"]
    dtype = DTYPES[case["dtype"]]
    if case["op"] == "append":
        return tuple(_values(_quantise(x.transpose(1, 2))).to(dtype) for x in (state["k"], state["v"]))
    if case["op"] == "read":
        return tuple(_values(x).to(dtype) for x in state["held"])
    k, v = (_values(x) for x in state["held"])  # [B, H, n, D]
    q = state["q"].float()
    b, t, qh, d = q.shape
    q = q.view(b, t, case["heads"], case["group"], d).permute(0, 2, 3, 1, 4).reshape(b, case["heads"], -1, d)
    s = torch.matmul(q, k.transpose(-1, -2)).view(b, case["heads"], case["group"], t, -1) / math.sqrt(d)
    at = state["starts"].view(b, 1, 1, 1, 1) + torch.arange(t, device=q.device).view(1, 1, 1, t, 1)
    s = s.masked_fill(torch.arange(s.shape[-1], device=q.device) > at, float("-inf"))
    p = (s - s.amax(-1, keepdim=True)).exp()
    p = (p / p.sum(-1, keepdim=True)).view(b, case["heads"], case["group"] * t, -1)
    o = torch.matmul(p, v).view(b, case["heads"], case["group"], t, d)
    return o.permute(0, 3, 1, 2, 4).reshape(b, t, qh * d).to(dtype)


def run(state):
    if not own:
        return _plain(state)
    from forgeml_b200.nebula import ops

    case = state["case"]
    if case["op"] == "append":
        ops.kv4_append(state["k"], state["v"], state["pool"], state["slot_of"], state["starts"])
        return ops.kv4_read(state["pool"], state["slot_of"], case["t"], start_pos=state["starts"])
    if case["op"] == "read":
        return ops.kv4_read(state["pool"], state["slot_of"], case["t"])
    return ops.kv4_attention(state["q"], state["pool"], state["slot_of"], state["starts"])


# ------------------------------------------------------------- the definition
def _stands_for(x):
    """What a row of numbers x [n, D] reads back as, in 64 bits, group by group."""
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    for c0 in range(0, x.shape[-1], GROUP):
        part = x[:, c0:c0 + GROUP].double()
        z = part.min(dim=1, keepdim=True).values
        s = ((part.max(dim=1, keepdim=True).values - z) / 15).to(x.dtype).double()
        quotient = (part - z) / torch.where(s == 0, torch.ones_like(s), s)
        code = torch.minimum(quotient.round(), torch.full_like(quotient, 15.0))
        out[:, c0:c0 + GROUP] = torch.where(s == 0, z, z + code * s)
    return out


def exact(case, seed):
    global own
    was, own = own, False
    try:
        dtype = DTYPES[case["dtype"]]
        dev = torch.device("cuda")
        b, t, h, d = case["batch"], case["t"], case["heads"], case["dim"]
        g = torch.Generator(device=dev)
        g.manual_seed(seed)
        torch.randperm(b + 2, generator=g, device=dev)
        starts = _starts(case)
        n = t if case["op"] != "attention" else max(starts) + t
        k, v = _rows(g, b, n, h, d, dtype)
        if case["op"] != "attention":
            out = tuple(torch.empty(b, h, n, d, dtype=torch.float64, device=dev) for _ in range(2))
            for x, y in zip((k, v), out):
                for i in range(b):
                    y[i] = _stands_for(x[i].reshape(n * h, d)).view(n, h, d).transpose(0, 1)
            return out
        q = torch.randn(b, t, h * case["group"], d, device=dev, dtype=dtype, generator=g)
        out = torch.empty(b, t, h * case["group"], d, dtype=torch.float64, device=dev)
        for i in range(b):
            m = starts[i] + t
            for j in range(h):
                kk, vv = _stands_for(k[i, :m, j]), _stands_for(v[i, :m, j])
                late = torch.ones(t, m, dtype=torch.bool, device=dev).triu(starts[i] + 1)
                for a in range(j * case["group"], (j + 1) * case["group"]):
                    s = (q[i, :, a].double() @ kk.T) * d ** -0.5
                    s[late] = -math.inf
                    out[i, :, a] = torch.softmax(s, dim=-1) @ vv
        return out.reshape(b, t, -1)
    finally:
        own = was
