"""What is timed of the gated recurrence and of dropout, with their plain forms.

Operators (yufmusicgen_b200/gated_scan.py, yufmusicgen_b200/dropout.py):

* gated scan, per channel of [B, T, D]:
      a_t = lower + (1 - lower) sigmoid(f_t)
      h_t = a_t h_{t-1} + (1 - a_t) x_t
      y_t = h_t sigmoid(g_t)               (y_t = h_t without a gate)
  from an initial state h_0 [B, D] (zeros without one), also over sequences of
  different lengths packed into one row (cu_seqlens), with its gradients;
* its single-token form, which updates the state in place;
* dropout (+ residual): y = residual + keep * x / (1 - p).  Element i is kept
  when word i % 4 of Philox4x32-10(key = seed, counter = (i / 4, step)) is at
  least floor(p 2^32); the backward pass draws the same words again.
"""

import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
MOST = 16 * 8192 * 1024  # elements of the largest case's tensors


def _scan(name, B, T, D, dtype, **kw):
    c = {"op": "scan", "B": B, "T": T, "D": D, "dtype": dtype, "train": False, "gate": True, "lower": True,
         "state": True, "seqs": 0, "fused": False}
    c.update(kw)
    return {"name": name, **c}


def _drop(name, rows, cols, dtype, residual, p, train):
    return {"name": name, "op": "dropout", "rows": rows, "cols": cols, "dtype": dtype, "residual": residual,
            "p": p, "train": train}


def listed():
    return [
        # prefill of two prompts through a layer of the 0.1B model: x, f and g are column ranges of one projection
        _scan("prefill 2x2048x640 bf16", 2, 2048, 640, "bf16", fused=True),
        # one long prompt: few channels in flight, the time axis has to be split
        _scan("prefill 1x16384x1024 bf16", 1, 16384, 1024, "bf16", state=False),
        # packed prompts of different lengths, some empty, an odd width, rows behind the last one
        _scan("prefill packed 10007x333 fp16", 1, 10007, 333, "fp16", seqs=37),
        # training step of the tiny configuration, where latency counts
        _scan("train 2x256x128 fp32", 2, 256, 128, "fp32", train=True, state=False),
        # training step of a layer of the 0.1B model
        _scan("train 8x2048x640 bf16", 8, 2048, 640, "bf16", train=True),
        # training on long sequences at d = 1024
        _scan("train 16x8192x1024 bf16", 16, 8192, 1024, "bf16", train=True, state=False),
        # training on packed pieces, one layer without the output gate, fp32
        _scan("train packed 12345x250 fp32", 1, 12345, 250, "fp32", train=True, gate=False, seqs=61),
        # one token of one sequence
        {"name": "step 1x640 bf16", "op": "step", "B": 1, "D": 640, "dtype": "bf16", "gate": True, "lower": True},
        # one token of each of 256 sequences (batched decode)
        {"name": "step 256x640 fp32", "op": "step", "B": 256, "D": 640, "dtype": "fp32", "gate": True, "lower": True},
        # the tiny configuration's block output
        _drop("dropout 512x128 fp32", 512, 128, "fp32", "none", 0.1, True),
        # block outputs in bf16 added to an fp32 residual stream, forward and backward
        _drop("dropout 131072x1024 bf16+fp32", 16 * 8192, 1024, "bf16", "fp32", 0.1, True),
        # an odd width, forward only
        _drop("dropout 10007x333 fp16+fp16", 10007, 333, "fp16", "same", 0.25, False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    op = rng.choice(["scan", "scan", "scan", "train", "train", "train", "step", "dropout", "dropout"])
    dtype = rng.choice(sorted(DTYPES))
    if op == "step":
        return {"op": "step", "B": _log(rng, 1, 1024), "D": _log(rng, 16, 1024), "dtype": dtype,
                "gate": rng.random() < 0.75, "lower": rng.random() < 0.75}
    if op == "dropout":
        cols = _log(rng, 16, 1024)
        rows = _log(rng, 1, min(131072, MOST // cols // 2))
        return {"op": "dropout", "rows": rows, "cols": cols, "dtype": dtype,
                "residual": rng.choice(["none", "same", "fp32"]), "p": round(rng.uniform(0.02, 0.6), 3),
                "train": rng.random() < 0.6}
    train = op == "train"
    packed = rng.random() < 0.35
    D = _log(rng, 16, 1024)
    B = 1 if packed else _log(rng, 1, 64)
    T = _log(rng, 1, 16384)
    T = max(1, min(T, MOST // 2 // (B * D)))
    return {"op": "scan", "B": B, "T": T, "D": D, "dtype": dtype, "train": train,
            "gate": rng.random() < 0.75, "lower": rng.random() < 0.75, "state": rng.random() < 0.6,
            "seqs": _log(rng, 1, 128) if packed else 0, "fused": (not train) and rng.random() < 0.5}


def prepare(case, seed):
    dev = "cuda"
    gen = torch.Generator(device=dev)
    gen.manual_seed(int(seed))
    dt = DTYPES[case["dtype"]]

    def rnd(*shape, scale=1.0, shift=0.0, dtype=None):
        t = torch.randn(*shape, generator=gen, device=dev, dtype=torch.float32)
        return t.mul_(scale).add_(shift).to(dtype or dt)

    def floors(D):  # retention floors: from forgetful channels to ones of long memory
        return torch.rand(D, generator=gen, device=dev) * 0.95

    if case["op"] == "dropout":
        shape = (case["rows"], case["cols"])
        rdt = {"none": None, "same": dt, "fp32": torch.float32}[case["residual"]]
        s = {"case": case, "x": rnd(*shape), "residual": None if rdt is None else rnd(*shape, dtype=rdt)}
        host = torch.Generator().manual_seed(int(seed))
        s["seed"], s["step"] = (int(torch.randint(0, 2**62, (), generator=host)) for _ in range(2))
        s["dy"] = rnd(*shape, dtype=rdt or dt) if case["train"] else None
        if case["train"]:
            s["x"].requires_grad_(True)
            if rdt is not None:
                s["residual"].requires_grad_(True)
        return s

    if case["op"] == "step":
        B, D = case["B"], case["D"]
        return {"case": case, "x": rnd(B, D), "f": rnd(B, D, scale=1.5, shift=2.0),
                "g": rnd(B, D) if case["gate"] else None, "lower": floors(D) if case["lower"] else None,
                "state": rnd(B, D, dtype=torch.float32)}

    B, T, D, n = case["B"], case["T"], case["D"], case["seqs"]
    s = {"case": case, "cu": None}
    if n:  # cut points anywhere, so some sequences are empty; a fiftieth of the rows lies behind the last one
        end = T - T // 50
        cuts = torch.randint(0, end + 1, (n - 1,), generator=gen, device=dev).sort().values
        s["cu"] = torch.cat([cuts.new_zeros(1), cuts, cuts.new_full((1,), end)]).to(torch.int32)
    x, f = rnd(B, T, D), rnd(B, T, D, scale=1.5, shift=2.0)
    g = rnd(B, T, D) if case["gate"] else None
    if case["fused"]:  # what one projection of the layer's input gives
        s["proj"] = torch.cat([t for t in (x, f, g) if t is not None], dim=-1)
    else:
        s["x"], s["f"], s["g"] = x, f, g
    rows = n or B
    s["lower"] = floors(D) if case["lower"] else None
    s["state"] = rnd(rows, D, dtype=torch.float32) if case["state"] else None
    if case["train"]:
        s["dy"], s["dh"] = rnd(B, T, D), rnd(rows, D, dtype=torch.float32)
        s["leaves"] = [t for t in (s["x"], s["f"], s["g"], s["lower"], s["state"]) if t is not None]
        for t in s["leaves"]:
            t.requires_grad_(True)
    return s


def _parts(state):
    """x, f and g of a pass: tensors of their own, or column ranges of one projection."""
    if "proj" in state:
        p = state["proj"].split(state["case"]["D"], dim=-1)
        return p[0], p[1], p[2] if len(p) > 2 else None
    return state["x"], state["f"], state["g"]


def run(state):
    case = state["case"]
    if case["op"] == "dropout":
        if own:
            from yufmusicgen_b200.dropout import dropout
            y = dropout(state["x"], case["p"], state["seed"], state["step"], residual=state["residual"])
            if not case["train"]:
                return {"y": y}
            leaves = [t for t in (state["x"], state["residual"]) if t is not None]
            grads = torch.autograd.grad(y, leaves, state["dy"])
            return {"y": y.detach(), "dx": grads[0], "dr": grads[1] if len(grads) > 1 else None}
        return _plain_dropout(state)
    if case["op"] == "step":
        if own:
            from yufmusicgen_b200.gated_scan import gated_scan_step
            y = gated_scan_step(state["x"], state["f"], state["state"], gate=state["g"], lower=state["lower"])
            return {"y": y, "state": state["state"]}
        return _plain_step(state)
    if own:
        from yufmusicgen_b200.gated_scan import gated_scan
        x, f, g = _parts(state)
        y, h = gated_scan(x, f, gate=g, lower=state["lower"], state=state["state"], cu_seqlens=state["cu"])
        if not case["train"]:
            return {"y": y, "h": h}
        grads = iter(torch.autograd.grad((y, h), state["leaves"], (state["dy"], state["dh"])))
        out = {"y": y.detach(), "h": h.detach(), "dx": next(grads), "df": next(grads)}
        out["dg"] = next(grads) if state["g"] is not None else None
        out["dlower"] = next(grads) if state["lower"] is not None else None
        out["dstate"] = next(grads) if state["state"] is not None else None
        return out
    with torch.no_grad():
        return _plain_scan(state)


# ---- plain forms: elementary operations, 32 bits inside, rounded once ----

def _sigmoid(v):
    return 1.0 / (1.0 + torch.exp(-v))


def _rates(f, lower):
    """sigmoid(f), the retention a and the input share 1 - a (without its cancellation)."""
    s, i = _sigmoid(f), _sigmoid(-f)
    if lower is None:
        return s, s, i
    return s, lower + (1.0 - lower) * s, (1.0 - lower) * i


def _doubling(a, b):
    """All prefixes of h_t = a_t h_{t-1} + b_t along dim 1, in log2(T) passes."""
    a, b, k, T = a.clone(), b.clone(), 1, a.shape[1]
    while k < T:
        b[:, k:] = b[:, k:] + a[:, k:] * b[:, :-k]
        a[:, k:] = a[:, k:] * a[:, :-k]
        k *= 2
    return b


def _owners(cu, T):
    """Row of cu_seqlens that each token belongs to, and where sequences start, end and live."""
    t = torch.arange(T, device=cu.device)
    seq = (t[:, None] >= cu[None, :]).sum(1) - 1
    live = (seq >= 0) & (seq < cu.numel() - 1)
    seq = seq.clamp(0, cu.numel() - 2)
    return seq, live, live & (t == cu[seq]), live & (t + 1 == cu[seq + 1])


def _plain_scan(state):
    case, (x, f, g), cu = state["case"], _parts(state), state["cu"]
    dt, (B, T, D) = x.dtype, x.shape
    lower, h0 = state["lower"], state["state"]
    xf = x.float()
    s, a, i = _rates(f.float(), lower)
    b = i * xf
    carry = a.clone()  # what each token takes over from the one before it in the same row
    if cu is None:
        carry[:, 0] = 0
        if h0 is not None:
            b[:, 0] = b[:, 0] + a[:, 0] * h0
    else:
        seq, live, first, last = _owners(cu, T)
        b = b * live[None, :, None]
        carry[:, first] = 0
        if h0 is not None:
            b[0, first] = b[0, first] + a[0, first] * h0[seq[first]]
    h = _doubling(carry, b)
    sg = 1.0 if g is None else _sigmoid(g.float())
    y = h * sg
    if cu is None:
        end = h[:, -1].clone()
    else:
        y = y * live[None, :, None]
        end = torch.zeros(cu.numel() - 1, D, device=x.device) if h0 is None else h0.clone()
        end[seq[last]] = h[0, last]
    out = {"y": y.to(dt), "h": end}
    if not case["train"]:
        return out
    # gradients: dh_t = dy_t sigmoid(g_t) + a_{t+1} dh_{t+1}
    dy, dend = state["dy"].float(), state["dh"]
    p = dy * sg
    if cu is None:
        p[:, -1] = p[:, -1] + dend
    else:
        p = p * live[None, :, None]
        p[0, last] = p[0, last] + dend[seq[last]]
    nxt = torch.zeros_like(carry)
    nxt[:, :-1] = carry[:, 1:]
    dh = _doubling(nxt.flip(1), p.flip(1)).flip(1)
    if cu is not None:
        dh = dh * live[None, :, None]
    prev = torch.zeros_like(h)
    prev[:, 1:] = h[:, :-1]
    if cu is None:
        prev[:, 0] = 0.0 if h0 is None else h0
    else:
        prev[0, first] = 0.0 if h0 is None else h0[seq[first]]
    da = dh * (prev - xf)
    out["dx"] = (dh * i).to(dt)
    out["df"] = (da * i * s).to(dt)
    if g is not None:
        dg = dy * h * sg * _sigmoid(-g.float())
        out["dg"] = (dg if cu is None else dg * live[None, :, None]).to(dt)
    else:
        out["dg"] = None
    out["dlower"] = None if lower is None else (da * _sigmoid(-f.float())).sum((0, 1), dtype=torch.float64).float()
    if h0 is None:
        out["dstate"] = None
    elif cu is None:
        out["dstate"] = a[:, 0] * dh[:, 0]
    else:
        ds = dend.clone()
        ds[seq[first]] = a[0, first] * dh[0, first]
        out["dstate"] = ds
    return out


def _plain_step(state):
    _, a, i = _rates(state["f"].float(), state["lower"])
    h = state["state"]
    h.copy_(a * h + i * state["x"].float())
    y = h if state["g"] is None else h * _sigmoid(state["g"].float())
    return {"y": y.to(state["x"].dtype), "state": h}


M32 = 0xFFFFFFFF


def _philox_words(n, seed, step, device):
    """The first n 32-bit words of the stream (int64 tensors hold them)."""
    q = torch.arange((n + 3) // 4, device=device, dtype=torch.int64)
    c0, c1 = q & M32, q >> 32
    c2, c3 = (torch.full_like(q, w) for w in (step & M32, (step >> 32) & M32))
    k0, k1 = seed & M32, (seed >> 32) & M32
    for _ in range(10):
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57  # the low 64 bits of the product: the sign does not matter
        c0, c1, c2, c3 = ((p1 >> 32) & M32) ^ c1 ^ k0, p1 & M32, ((p0 >> 32) & M32) ^ c3 ^ k1, p0 & M32
        k0, k1 = (k0 + 0x9E3779B9) & M32, (k1 + 0xBB67AE85) & M32
    return torch.stack([c0, c1, c2, c3], dim=1).reshape(-1)[:n]


def _plain_dropout(state):
    case = state["case"]
    with torch.no_grad():
        x, r = state["x"], state["residual"]
        keep = (_philox_words(x.numel(), state["seed"], state["step"], x.device) >= int(case["p"] * 2**32)).reshape(x.shape)
        scale = 1.0 / (1.0 - case["p"])
        y = torch.where(keep, x.float() * scale, 0.0)
        out = {"y": y.to(x.dtype) if r is None else (r.float() + y).to(r.dtype)}
        if case["train"]:
            out["dx"] = torch.where(keep, state["dy"].float() * scale, 0.0).to(x.dtype)
            out["dr"] = None if r is None else state["dy"]
        return out


# ---- the definitions in 64 bits, token by token ----

def exact(case, seed):
    with torch.no_grad():
        s = prepare(case, seed)
        if case["op"] == "dropout":
            return _exact_dropout(case, s)
        if case["op"] == "step":
            h, y = _exact_token(s["x"].double(), s["f"].double(), s["g"], s["lower"], s["state"].double())
            return {"y": y, "state": h}
        return _exact_scan(case, s)


def _exact_token(x, f, g, lower, h):
    low = 0.0 if lower is None else lower.double()
    share = (1.0 - low) / (1.0 + torch.exp(f))
    h = h + share * (x - h)
    return h, h if g is None else h / (1.0 + torch.exp(-g.double()))


def _exact_scan(case, s):
    x, f, g = (None if t is None else t.detach().double() for t in _parts(s))
    B, T, D = x.shape
    low = torch.zeros(D, device=x.device, dtype=torch.float64) if s["lower"] is None else s["lower"].double()
    share = (1.0 - low) / (1.0 + torch.exp(f))  # 1 - a
    rows = case["seqs"] or B
    start = torch.zeros(rows, D, device=x.device, dtype=torch.float64) if s["state"] is None else s["state"].double()
    pieces = [(None, 0, T)] if s["cu"] is None else []
    if s["cu"] is not None:
        cu = s["cu"].tolist()
        pieces = [(n, cu[n], cu[n + 1]) for n in range(rows)]
    hist, before = torch.zeros_like(x), torch.zeros_like(x)
    end = start.clone()
    for n, lo, hi in pieces:
        h = start if n is None else start[n:n + 1]
        for t in range(lo, hi):
            before[:, t] = h
            h = torch.lerp(h, x[:, t], share[:, t])
            hist[:, t] = h
        if n is None:
            end = h.clone()
        else:
            end[n] = h[0]
    sg = None if g is None else 1.0 / (1.0 + torch.exp(-g))
    out = {"y": hist if g is None else hist * sg, "h": end}
    if not case["train"]:
        return out
    dy = s["dy"].double()
    p = dy if g is None else dy * sg
    dhist, dstart = torch.zeros_like(x), s["dh"].double().clone()
    for n, lo, hi in pieces:
        c = s["dh"].double() if n is None else s["dh"][n:n + 1].double()
        for t in range(hi - 1, lo - 1, -1):
            c = c + p[:, t]
            dhist[:, t] = c
            c = c - c * share[:, t]
        if n is None:
            dstart = c
        else:
            dstart[n] = c[0]
    out["dx"] = dhist * share
    dsig = dhist * (before - x)  # gradient of a
    keep = 1.0 / (1.0 + torch.exp(-f))
    out["df"] = dsig * (1.0 - low) * keep / (1.0 + torch.exp(f))
    if g is not None:
        dg = dy * hist * sg * (1.0 / (1.0 + torch.exp(g)))
        if pieces and pieces[-1][0] is not None:
            dg[:, pieces[-1][2]:] = 0
        out["dg"] = dg
    else:
        out["dg"] = None
    out["dlower"] = None if s["lower"] is None else (dsig / (1.0 + torch.exp(f))).sum((0, 1))
    out["dstate"] = None if s["state"] is None else dstart
    return out


def _mul32(a, m):
    """High and low words of a 32 x 32-bit product, from 16-bit halves."""
    ah, al, mh, ml = a >> 16, a & 0xFFFF, m >> 16, m & 0xFFFF
    ll, lh, hl = al * ml, al * mh, ah * ml
    mid = (ll >> 16) + (lh & 0xFFFF) + (hl & 0xFFFF)
    return ah * mh + (lh >> 16) + (hl >> 16) + (mid >> 16), ((mid & 0xFFFF) << 16) | (ll & 0xFFFF)


def _exact_dropout(case, s):
    x = s["x"].detach().reshape(-1)
    n = x.numel()
    keep = torch.empty(n, dtype=torch.bool, device=x.device)
    limit = math.floor(case["p"] * 4294967296.0)
    part = 1 << 22  # counters at a time
    for q0 in range(0, (n + 3) // 4, part):
        q = torch.arange(q0, min(q0 + part, (n + 3) // 4), device=x.device)
        ctr = [q % 2**32, q // 2**32, torch.full_like(q, s["step"] % 2**32), torch.full_like(q, s["step"] // 2**32)]
        for r in range(10):
            key = (s["seed"] % 2**32 + r * 0x9E3779B9) % 2**32, (s["seed"] // 2**32 + r * 0xBB67AE85) % 2**32
            h0, l0 = _mul32(ctr[0], 0xD2511F53)
            h1, l1 = _mul32(ctr[2], 0xCD9E8D57)
            ctr = [h1 ^ ctr[1] ^ key[0], l1, h0 ^ ctr[3] ^ key[1], l0]
        for w in range(4):
            at = keep[4 * q0 + w:min(4 * (q0 + part), n):4]
            at.copy_(ctr[w][:at.numel()] >= limit)
    keep = keep.reshape(s["x"].shape)
    up = 1.0 - case["p"]
    y = torch.where(keep, s["x"].detach().double() / up, 0.0)
    out = {"y": y if s["residual"] is None else y + s["residual"].detach().double()}
    if case["train"]:
        out["dx"] = torch.where(keep, s["dy"].double() / up, 0.0)
        out["dr"] = None if s["residual"] is None else s["dy"].double()
    return out


def work(case):
    e = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "dropout":
        n = case["rows"] * case["cols"]
        r = {"none": 0, "same": e, "fp32": 4}[case["residual"]]
        out = r or e
        bytes_ = n * (e + r + out)  # x, residual, y
        if case["train"]:
            bytes_ += n * (out + e)  # dy, dx (the residual's gradient is dy)
        return {"bytes": bytes_, "flops": 2 * n}
    if case["op"] == "step":
        n = case["B"] * case["D"]
        return {"bytes": n * (e * (3 + case["gate"]) + 8) + 4 * case["D"] * case["lower"], "flops": 14 * n}
    n, rows = case["B"] * case["T"] * case["D"], (case["seqs"] or case["B"]) * case["D"]
    small = 4 * rows * (1 + case["state"]) + 4 * case["D"] * case["lower"]
    if not case["train"]:
        return {"bytes": n * e * (3 + case["gate"]) + small, "flops": 14 * n}
    # x, f, g, dy read; y, dx, df, dg written
    return {"bytes": n * e * (6 + 2 * case["gate"]) + 2 * small, "flops": 40 * n}
