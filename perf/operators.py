"""Attention between ragged sets of an event, and what prepares its queries and keys, as timed cases.

``CrossAttention``: the rows of one ragged batch (hits, or a few object queries per event) attend to the
rows of another one of the same events (condensates, or all hits), forward and with its gradients.
``NormRotate``: the normalisation of queries and keys per head with the rotation by their positions (hit
coordinates, or the place in the event), forward and with its gradients.

Event sizes are those of the benchmark configurations and of the test suite: 700 hits as an online service
sees them, 1500 to 31000 in small ragged batches, 50k to 150k in the batch of four, 200k in full events.
"""
import math

import torch

own = False

_TYPES = {"float": torch.float32, "half": torch.float16, "bfloat": torch.bfloat16}
_EPS = 1e-6


# ------------------------------------------------------------------------------------------- cases
def _attend(events, queries, keys, heads, kv_heads, dim, dtype, masked=False, packed=False, train=False):
    """Between ``events`` events with ``queries`` = (fewest, most) rows each and ``keys`` likewise.  ``masked``: a tenth
    of the keys is noise that no query may see.  ``packed``: keys and values are views of one projection's result."""
    return dict(kind="attend", events=events, q_lo=queries[0], q_hi=queries[1], k_lo=keys[0], k_hi=keys[1], heads=heads,
                kv_heads=kv_heads, dim=dim, dtype=dtype, masked=masked, packed=packed, train=train)


def _rotate(queries, keys, heads, kv_heads, dim, rotary, axes, dtype, interleaved=False, packed=False, train=False):
    """``queries`` and ``keys`` rows (no keys: queries alone), of which ``rotary`` columns turn with ``axes`` coordinates
    (0: with the integer place in the event)."""
    return dict(kind="rotate", queries=queries, keys=keys, heads=heads, kv_heads=kv_heads, dim=dim, rotary=rotary,
                axes=axes, dtype=dtype, interleaved=interleaved, packed=packed, train=train)


def listed():
    named = [
        # an online service: one new query looks at the hits of one small event; launches and latency count
        ("attend_one_query_700", _attend(1, (1, 1), (700, 700), 8, 8, 64, "bfloat")),
        # one query per event looks at the kept keys and values of a large ragged batch, four heads to a key head
        ("attend_query_per_event_64", _attend(64, (1, 1), (200, 40000), 8, 2, 64, "bfloat")),
        # a few hundred object queries per event read the hits of four mid-size events, noise left out
        ("attend_objects_to_hits", _attend(4, (100, 400), (50000, 150000), 8, 8, 32, "bfloat", masked=True, packed=True)),
        # every hit reads the condensates of its event
        ("attend_hits_to_objects", _attend(4, (50000, 150000), (100, 400), 4, 4, 64, "half")),
        # small ragged events in the library's own type, a width that is no multiple of a vector
        ("attend_odd_ragged", _attend(7, (1500, 31000), (300, 5000), 3, 1, 22, "float")),
        # a training step on a few small events in the library's own type
        ("attend_train_small", _attend(3, (5000, 9000), (1000, 3001), 4, 4, 32, "float", masked=True, train=True)),
        # a training step between the hits of two views of an event: the largest amount of work
        ("attend_train_hits", _attend(4, (5000, 31000), (5000, 31000), 8, 8, 64, "bfloat", train=True)),
        # wide heads, two to a key head, on one full-size event
        ("attend_train_wide_200k", _attend(1, (200000, 200000), (1000, 1000), 4, 2, 128, "half", packed=True, train=True)),
        # the new query of an online service gets its norm and its rotation
        ("rotate_one_query", _rotate(1, 0, 8, 8, 64, 64, 0, "bfloat")),
        # object queries and the hits of four mid-size events, turned with four coordinates
        ("rotate_objects_and_hits", _rotate(1000, 400000, 8, 8, 32, 32, 4, "bfloat", packed=True)),
        # odd sizes in the library's own type: some columns are not turned, neighbouring columns form pairs
        ("rotate_odd", _rotate(20011, 7013, 3, 1, 22, 12, 3, "float", interleaved=True)),
        # a training step on one full-size event
        ("rotate_train_200k", _rotate(200000, 200000, 8, 2, 64, 64, 0, "bfloat", train=True)),
    ]
    return [dict(c, name=n) for n, c in named]


def draw(rng):
    def log_int(a, b):
        return int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))

    dtype = rng.choice(["bfloat", "bfloat", "half", "float"])
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    heads = kv_heads * rng.choice([1, 1, 1, 2, 3, 4])
    dim = rng.choice([8, 16, 22, 32, 32, 40, 64, 64, 64, 72, 96, 128, 128, rng.randint(4, 128)])
    train = rng.random() < 0.5
    if rng.random() < 0.65:
        # 9e9 pairs of rows and heads at most, a twelfth of it in float32 and for widths that are no whole vectors
        most = 6e11 / (12 if dtype == "float" or dim % 8 else 1) / (heads * max(dim, 64))
        total_q, total_k = log_int(1, 200000), log_int(1, 400000)
        events = min(log_int(1, 64), max(total_q, total_k))
        while total_q * total_k / events > most:
            total_q, total_k = max(1, int(total_q * 0.8)), max(1, int(total_k * 0.8))
        spread = rng.choice([0., 0.3, 0.9, 1.])
        ends = []
        for total in (total_q, total_k):
            mean = total / events
            lo = int(mean * (1 - spread))
            ends.append((lo, max(1, lo, int(mean * (1 + spread)) + rng.randint(0, 3))))
        return _attend(events, ends[0], ends[1], heads, kv_heads, dim, dtype, masked=rng.random() < 0.4,
                       packed=rng.random() < 0.4, train=train)
    axes = rng.choice([0, 0, 1, 2, 3, 4])
    step = 2 * max(axes, 1)
    dim = max(dim, step)
    rotary = dim // step * step if rng.random() < 0.7 else step * rng.randint(1, dim // step)
    most = 1.0e8 / dim / (2 if dtype == "float" else 1)
    queries, keys = log_int(1, 200000), log_int(1, 400000) if rng.random() < 0.8 else 0
    while queries * heads + keys * kv_heads > most:
        queries, keys = max(1, int(queries * 0.8)), int(keys * 0.8)
    return _rotate(queries, keys, heads, kv_heads, dim, rotary, axes, dtype, interleaved=rng.random() < 0.4,
                   packed=rng.random() < 0.4, train=train)


# ------------------------------------------------------------------------------------------ inputs
def _sizes(events, lo, hi, phase):
    """Rows per event: spread over lo .. hi, in an order without a pattern."""
    return [lo + int((hi - lo + 1) * ((i * 0.6180339887 + phase) % 1.0)) for i in range(events)]


def _event_sizes(case):
    return (_sizes(case["events"], case["q_lo"], case["q_hi"], 0.5),
            _sizes(case["events"], case["k_lo"], case["k_hi"], 0.7))


def _splits(sizes):
    out = [0]
    for n in sizes:
        out.append(out[-1] + n)
    return out


def _pair(n, heads, dim, dtype, packed, gen, std):
    """Two tensors [n, heads, dim]; packed: views of the rows of one buffer."""
    both = (torch.randn((n, 2, heads, dim), generator=gen, device=gen.device) * std).to(dtype)
    return (both[:, 0], both[:, 1]) if packed else (both[:, 0].contiguous(), both[:, 1].contiguous())


def _positions(n, axes, gen):
    """Coordinates in cm, as the hits of showers have them; without axes the place in an event that starts far on."""
    if axes:
        centres = 150. * (2. * torch.rand((300, axes), generator=gen, device=gen.device) - 1.)
        of = torch.randint(0, 300, (n,), generator=gen, device=gen.device)
        return centres[of] + 3. * torch.randn((n, axes), generator=gen, device=gen.device)
    start = torch.randint(0, 200000, (1,), generator=gen, device=gen.device)
    return (torch.arange(n, device=gen.device) + start).to(torch.int32)


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    dtype, heads, kv_heads, dim = _TYPES[case["dtype"]], case["heads"], case["kv_heads"], case["dim"]
    s = dict(case=case)
    if case["kind"] == "attend":
        nq, nk = _event_sizes(case)
        s["q_splits"], s["k_splits"] = _splits(nq), _splits(nk)
        s["rs_q"] = torch.tensor(s["q_splits"], dtype=torch.int32, device=dev)
        s["rs_k"] = torch.tensor(s["k_splits"], dtype=torch.int32, device=dev)
        s["q"] = torch.randn((sum(nq), heads, dim), generator=gen, device=dev).to(dtype)
        s["k"], s["v"] = _pair(sum(nk), kv_heads, dim, dtype, case["packed"], gen, 1.)
        s["mask"] = torch.rand((sum(nk),), generator=gen, device=dev) >= 0.1 if case["masked"] else None
        if case["train"]:
            s["grad"] = torch.randn(s["q"].shape, generator=gen, device=dev).to(dtype)
            for name in ("q", "k", "v"):
                s[name] = s[name].detach().requires_grad_(True)
        return s
    # activations of a projection have no unit size yet
    if case["packed"]:
        buf = (3. * torch.randn((case["queries"], heads + 1, dim), generator=gen, device=dev)).to(dtype)
        s["q"] = buf[:, :heads]
    else:
        s["q"] = (3. * torch.randn((case["queries"], heads, dim), generator=gen, device=dev)).to(dtype)
    s["wq"] = (1. + 0.2 * torch.randn((dim,), generator=gen, device=dev)).to(dtype)
    s["pq"] = _positions(case["queries"], case["axes"], gen)
    s["k"] = s["wk"] = s["pk"] = None
    if case["keys"]:
        s["k"], _ = _pair(case["keys"], kv_heads, dim, dtype, case["packed"], gen, 3.)
        s["wk"] = (1. + 0.2 * torch.randn((dim,), generator=gen, device=dev)).to(dtype)
        s["pk"] = _positions(case["keys"], case["axes"], gen)
    if case["train"]:
        for name in ("q", "k"):
            if s[name] is not None:
                s["g" + name] = torch.randn(s[name].shape, generator=gen, device=dev).to(dtype)
                s[name] = s[name].detach().requires_grad_(True)
                s["w" + name] = s["w" + name].requires_grad_(True)
    return s


# ------------------------------------------------------------------------------------- plain forms
def _by_event(s):
    """(rows of the queries, indices of the keys that they may see) of every event."""
    for e in range(s["case"]["events"]):
        lo, hi = s["k_splits"][e], s["k_splits"][e + 1]
        keys = torch.arange(lo, hi, device=s["q"].device)
        if s["mask"] is not None:
            keys = keys[s["mask"][lo:hi]]
        yield slice(s["q_splits"][e], s["q_splits"][e + 1]), keys


def _plain_attend(s):
    q, k, v = (s[name].detach() for name in ("q", "k", "v"))
    (nq, heads, dim), kv_heads = q.shape, k.shape[1]
    group, scale, train = heads // kv_heads, dim ** -0.5, s["case"]["train"]
    out = torch.zeros(q.shape, device=q.device)
    if train:
        dq, dk, dv = (torch.zeros(t.shape, device=q.device) for t in (q, k, v))

    def rows(t, a, b):  # [key heads, rows x heads of the group, dim]
        return t[a:b].float().reshape(b - a, kv_heads, group, dim).transpose(0, 1).reshape(kv_heads, (b - a) * group, dim)

    def back(t):
        return t.reshape(kv_heads, -1, group, dim).transpose(0, 1).reshape(-1, heads, dim)

    for event, keys in _by_event(s):
        if keys.numel() == 0:
            continue
        ke, ve = k[keys].float().transpose(0, 1), v[keys].float().transpose(0, 1)
        step = max(1, 200000000 // (heads * keys.numel()))
        for a in range(event.start, event.stop, step):
            b = min(a + step, event.stop)
            qe = rows(q, a, b)
            p = qe @ ke.transpose(1, 2)
            p = torch.exp((p - p.amax(-1, keepdim=True)) * scale)
            p = p / p.sum(-1, keepdim=True)
            out[a:b] = back(p @ ve)
            if train:
                ge = rows(s["grad"], a, b)
                dv[keys] += (p.transpose(1, 2) @ ge).transpose(0, 1)
                ds = ge @ ve.transpose(1, 2)
                ds = p * (ds - (p * ds).sum(-1, keepdim=True)) * scale
                dq[a:b] = back(ds @ ke)
                dk[keys] += (ds.transpose(1, 2) @ qe).transpose(0, 1)
    if not train:
        return out.to(q.dtype)
    return tuple(t.to(q.dtype) for t in (out, dq, dk, dv))


def _angles(positions, rotary, axes):
    """[rows, axes, pairs of an axis], in 64 bits: the integer part of a far angle leaves 32 few digits."""
    pairs = rotary // max(axes, 1) // 2
    freq = 10000. ** (-torch.arange(pairs, dtype=torch.float64, device=positions.device) / pairs)
    return positions.double().reshape(positions.shape[0], max(axes, 1), 1) * freq


def _turn(x, cos, sin, rotary, interleaved):
    """Turns the pairs of the leading ``rotary`` columns of [rows, heads, dim]."""
    n, heads, _ = x.shape
    axes, pairs = cos.shape[1], cos.shape[2]
    head = x[..., :rotary].reshape(n, heads, axes, *((pairs, 2) if interleaved else (2, pairs)))
    first, second = head.unbind(-1 if interleaved else -2)
    cos, sin = cos[:, None], sin[:, None]
    head = torch.stack((first * cos - second * sin, second * cos + first * sin), -1 if interleaved else -2)
    return torch.cat((head.reshape(n, heads, rotary), x[..., rotary:]), -1)


def _plain_rotate(s):
    c = s["case"]
    outs, grads, weights = [], [], []
    for name in ("q", "k"):
        if s[name] is None:
            continue
        x, w = s[name].detach().float(), s["w" + name].detach().float()
        angle = _angles(s["p" + name], c["rotary"], c["axes"])
        cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
        r = torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS)
        outs.append(_turn(x * r * w, cos, sin, c["rotary"], c["interleaved"]).to(s[name].dtype))
        if c["train"]:
            g = _turn(s["g" + name].float(), cos, -sin, c["rotary"], c["interleaved"])
            weights.append((g * x * r).sum((0, 1), dtype=torch.float64).to(s[name].dtype))
            g = g * w
            grads.append((r * (g - x * (r * r) * (g * x).mean(-1, keepdim=True))).to(s[name].dtype))
    return tuple(outs + grads + weights)


# ------------------------------------------------------------------------------------------- calls
def _own_attend(s):
    from hgcalml_b200.cross_attention_op import CrossAttention
    out = CrossAttention(s["q"], s["k"], s["v"], s["rs_q"], s["rs_k"], key_mask=s["mask"])
    if not s["case"]["train"]:
        return out
    return (out.detach(),) + torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["grad"])


def _own_rotate(s):
    from hgcalml_b200.norm_rotate_op import NormRotate
    c = s["case"]
    q, k = NormRotate(s["q"], s["k"], s["wq"], s["wk"], s["pq"], s["pk"], rotary_dim=c["rotary"],
                      interleaved=c["interleaved"], eps=_EPS)
    if not c["train"]:
        return (q,) if k is None else (q, k)
    if k is None:
        return (q.detach(),) + torch.autograd.grad(q, (s["q"], s["wq"]), s["gq"])
    return (q.detach(), k.detach()) + torch.autograd.grad((q, k), (s["q"], s["k"], s["wq"], s["wk"]), (s["gq"], s["gk"]))


def run(s):
    if s["case"]["kind"] == "attend":
        return _own_attend(s) if own else _plain_attend(s)
    return _own_rotate(s) if own else _plain_rotate(s)


# -------------------------------------------------------------------------------------------- work
def work(case):
    """Inputs read once, outputs written once; the products of attention with a row's keys (two forward, and four for
    the gradients), the operations of norm and rotation per element."""
    size = 4 if case["dtype"] == "float" else 2
    heads, kv_heads, dim, train = case["heads"], case["kv_heads"], case["dim"], case["train"]
    if case["kind"] == "attend":
        nq, nk = _event_sizes(case)
        pairs = sum(a * b for a, b in zip(nq, nk)) * (0.9 if case["masked"] else 1.)
        q, kv = sum(nq) * heads * dim * size, 2 * sum(nk) * kv_heads * dim * size
        both = 8 * (case["events"] + 1) + (sum(nk) if case["masked"] else 0)
        # forward: q, k, v, result; backward besides: gradient of the result, gradients of q, k, v
        return {"bytes": 2 * q + kv + both + (2 * q + kv if train else 0),
                "flops": int(2 * pairs * heads * dim * (6 if train else 2))}
    elements = (case["queries"] * heads + case["keys"] * kv_heads) * dim
    positions = (case["queries"] + case["keys"]) * 4 * max(case["axes"], 1)
    weights = (2 if case["keys"] else 1) * dim * size
    return {"bytes": elements * size * (4 if train else 2) + positions + weights * (2 if train else 1),
            "flops": elements * (22 if train else 8)}


# ------------------------------------------------------------------------------------------- exact
def _exact_attend(s):
    q, k, v = (s[name].detach() for name in ("q", "k", "v"))
    heads, kv_heads, dim, train = q.shape[1], k.shape[1], q.shape[2], s["case"]["train"]
    res = [torch.zeros(q.shape, dtype=torch.float64, device=q.device)]
    if train:
        res += [torch.zeros(t.shape, dtype=torch.float64, device=q.device) for t in (q, k, v)]
    for event, keys in _by_event(s):
        if keys.numel() == 0:
            continue
        step = max(1, 60000000 // keys.numel())
        for h in range(heads):
            kv = h // (heads // kv_heads)
            kh, vh = k[keys, kv].double(), v[keys, kv].double()
            for a in range(event.start, event.stop, step):
                part = slice(a, min(a + step, event.stop))
                qh = q[part, h].double()
                score = torch.mm(qh, kh.t()).div_(math.sqrt(dim))
                share = score.sub_(torch.logsumexp(score, 1, keepdim=True)).exp_()
                oh = torch.mm(share, vh)
                res[0][part, h] = oh
                if train:
                    gh = s["grad"][part, h].double()
                    # d/ds of softmax: share * (g.v - g.o)
                    slope = torch.mm(gh, vh.t()).sub_((gh * oh).sum(1, keepdim=True)).mul_(share).div_(math.sqrt(dim))
                    res[1][part, h] = torch.mm(slope, kh)
                    res[2][:, kv].index_add_(0, keys, torch.mm(slope.t(), qh))
                    res[3][:, kv].index_add_(0, keys, torch.mm(share.t(), gh))
    return tuple(res) if train else res[0]


def _exact_rotate(s):
    c = s["case"]
    rotary, axes, train = c["rotary"], max(c["axes"], 1), c["train"]
    pairs = rotary // (2 * axes)
    outs, inputs, weights, grads = [], [], [], []
    for name in ("q", "k"):
        if s[name] is None:
            continue
        x = s[name].detach().double().requires_grad_(train)
        w = s["w" + name].detach().double().requires_grad_(train)
        with torch.set_grad_enabled(train):
            y = x / torch.sqrt(x.square().mean(-1, keepdim=True) + _EPS) * w
            # a pair of columns is a complex number, the rotation a factor of modulus one
            place = torch.arange(rotary, device=x.device).reshape(axes, -1)
            first, second = (place[:, 0::2], place[:, 1::2]) if c["interleaved"] else (place[:, :pairs], place[:, pairs:])
            theta = s["p" + name].double().reshape(-1, axes)[:, :, None] / torch.pow(
                torch.tensor(10000., dtype=torch.float64, device=x.device),
                torch.arange(pairs, device=x.device, dtype=torch.float64) * 2 / (rotary // axes))
            z = torch.complex(y[..., first], y[..., second]) * torch.polar(torch.ones_like(theta), theta)[:, None]
            z = z.flatten(-2)
            y = y.clone().index_copy(2, first.flatten(), z.real).index_copy(2, second.flatten(), z.imag)
        outs.append(y)
        inputs.append(x)
        weights.append(w)
        if train:
            grads.append(s["g" + name].double())
    if not train:
        return tuple(outs)
    return tuple(o.detach() for o in outs) + torch.autograd.grad(outs, inputs + weights, grads)


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_attend(s) if case["kind"] == "attend" else _exact_rotate(s)
