"""Workloads of the sequence operators: the short causal convolution, the selective state space scan
and the residual norm, over prompts, single tokens and training passes.

``listed()`` names them, ``draw(rng)`` gives more of the same ranges, ``prepare(case, seed)`` makes
the inputs, ``run(state)`` is one pass and ``work(case)`` its bytes and operations.  ``run`` computes
the operators from their formulas with elementary torch operations, or, where ``own`` is true, with
the plans of ``nengo_ocl_b200.cura_sequence``.  ``exact`` evaluates the definitions in 64 bits.

Sequences of different lengths lie one after the other in one packed (tokens, channels) tensor; a
case gives their lengths as text.  ``op`` is ``conv``, ``scan`` or ``norm``; ``train`` adds the
backward pass.
"""

import math

import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_EPS = 1e-5


def listed():
    return [
        # one token of one sequence: the smallest call, where latency counts
        dict(name="conv_token", op="conv", dtype="f32", lengths="1", channels=1024, taps=4, silu=True, carry=True,
             train=False),
        # a batch of prompts of different lengths (one of them empty), state carried on
        dict(name="conv_prompts", op="conv", dtype="bf16", lengths="2048,1,777,4096,0,1270", channels=4096, taps=4,
             silu=True, carry=True, train=False),
        # a training step's convolution
        dict(name="conv_train", op="conv", dtype="f32", lengths="1023,1025,2048", channels=2048, taps=4, silu=True,
             carry=False, train=True),
        # one token of one sequence
        dict(name="scan_token", op="scan", dtype="f32", lengths="1", channels=1024, states=16, groups=1, gate=True,
             carry=True, train=False),
        # one token of each of many sequences: the state is all of the traffic
        dict(name="scan_tokens", op="scan", dtype="bf16", lengths=",".join(["1"] * 256), channels=4096, states=16,
             groups=1, gate=True, carry=True, train=False),
        # a batch of prompts
        dict(name="scan_prompts", op="scan", dtype="f32", lengths="1024,2048,512,513", channels=4096, states=16,
             groups=1, gate=True, carry=True, train=False),
        # one long prompt of a narrow model: few channels, a long time axis
        dict(name="scan_long", op="scan", dtype="bf16", lengths="16384", channels=1024, states=16, groups=1, gate=True,
             carry=True, train=False),
        # a training step's scan
        dict(name="scan_train", op="scan", dtype="f32", lengths="2048,2048", channels=2048, states=16, groups=1,
             gate=True, carry=False, train=True),
        # the same with ragged lengths, odd sizes, groups and a 16-bit type
        dict(name="scan_train_odd", op="scan", dtype="f16", lengths="1000,3,517,1,0,2100", channels=1010, states=12,
             groups=2, gate=True, carry=True, train=True),
        # one token of a few sequences
        dict(name="norm_tokens", op="norm", dtype="f32", lengths="4", channels=1024, groups=1, gate="first",
             train=False),
        # the rows of a prompt
        dict(name="norm_prompt", op="norm", dtype="bf16", lengths="8192", channels=4096, groups=1, gate="first",
             train=False),
        # a training step's rows, norms over groups of channels
        dict(name="norm_train", op="norm", dtype="bf16", lengths="4096", channels=4096, groups=8, gate="first",
             train=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw_lengths(rng, total):
    """Between one and nine sequences with ``total`` tokens in all; sometimes one is empty."""
    n = min(rng.randint(1, 9), total)
    cuts = sorted(rng.sample(range(1, total), n - 1)) if n > 1 else []
    lengths = [b - a for a, b in zip([0] + cuts, cuts + [total])]
    if rng.random() < 0.3:
        lengths.insert(rng.randrange(len(lengths) + 1), 0)
    return ",".join(map(str, lengths))


def draw(rng):
    op = rng.choice(["conv", "scan", "scan", "norm"])
    train = rng.random() < 0.4
    case = dict(op=op, dtype=rng.choice(["f32", "f16", "bf16"]), train=train)
    channels = _log_int(rng, 64, 4096)
    if rng.random() < 0.6:
        channels = max(64, channels // 64 * 64)
    tokens = not train and rng.random() < 0.3
    if op == "conv":
        case.update(channels=channels, taps=rng.choice([2, 3, 4, 4, 4, 5, 8]), silu=rng.random() < 0.8,
                    carry=rng.random() < 0.7)
        limit = 33_000_000 // (4 if train else 1)
    elif op == "scan":
        groups = rng.choice([1, 1, 2, 4])
        case.update(channels=max(1, channels // groups) * groups, groups=groups,
                    states=rng.choice([3, 4, 8, 12, 16, 16, 16, 16, 32, 64]), gate=rng.random() < 0.8,
                    carry=rng.random() < 0.7)
        limit = (60_000_000 if train else 260_000_000) // case["states"]
    else:
        groups = rng.choice([1, 1, 2, 8])
        case.update(channels=max(1, channels // groups) * groups, groups=groups,
                    gate=rng.choice(["first", "last", "none"]))
        limit = 33_000_000 // (2 if train else 1)
    if tokens:
        case["lengths"] = ",".join(["1"] * _log_int(rng, 1, 256))
    else:
        case["lengths"] = _draw_lengths(rng, _log_int(rng, 16, min(4096 if train else 16384, limit // case["channels"])))
    return case


def _lengths(case):
    return [int(v) for v in case["lengths"].split(",")]


# ---- inputs ----------------------------------------------------------------------------------


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    dtype, lengths, chan = _TYPES[case["dtype"]], _lengths(case), case["channels"]
    total, n_seq = sum(lengths), len(lengths)

    def normal(*shape, scale=1.0, dtype=dtype):
        return (torch.randn(*shape, generator=gen, device=dev) * scale).to(dtype)

    def uniform(*shape, lo, hi):
        return torch.rand(*shape, generator=gen, device=dev) * (hi - lo) + lo

    f32 = torch.float32
    s = dict(case=case, lengths=lengths, x=normal(total, chan))
    if case["op"] == "conv":
        taps = case["taps"]
        s.update(w=uniform(chan, taps, lo=-taps ** -0.5, hi=taps ** -0.5), bias=normal(chan, scale=0.1, dtype=f32))
        if case["carry"]:
            s["state"] = normal(n_seq, taps - 1, chan)
        if case["train"]:
            s["dy"] = normal(total, chan)
            if case["carry"]:
                s["dnew_state"] = normal(n_seq, taps - 1, chan)
    elif case["op"] == "scan":
        groups, n = case["groups"], case["states"]
        # step sizes are log-uniform in [0.001, 0.1] after the softplus, decay rates around 1..n
        step = torch.exp(uniform(chan, lo=math.log(1e-3), hi=math.log(1e-1)))
        s.update(dt=normal(total, chan, scale=0.5), dt_bias=step + torch.log(-torch.expm1(-step)),
                 A=-torch.arange(1, n + 1, device=dev, dtype=f32) * uniform(chan, n, lo=0.7, hi=1.4),
                 B=normal(total, groups * n), C=normal(total, groups * n, scale=n ** -0.5),
                 D=uniform(chan, lo=0.5, hi=1.5))
        if case["gate"]:
            s["z"] = normal(total, chan)
        if case["carry"]:
            s["state"] = normal(n_seq, chan, n, scale=0.3, dtype=f32)
        if case["train"]:
            s["dy"] = normal(total, chan)
            if case["carry"]:
                s["dnew_state"] = normal(n_seq, chan, n, scale=0.1, dtype=f32)
    else:
        s.update(residual=normal(total, chan), weight=uniform(chan, lo=0.5, hi=1.5),
                 norm_weight=uniform(chan, lo=0.5, hi=1.5), scale=uniform(chan, lo=0.2, hi=0.6))
        if case["gate"] != "none":
            s["gate"] = normal(total, chan)
        if case["train"]:
            s.update(dy=normal(total, chan), dh=normal(total, chan))
    s.update(_index(case, lengths, dev))
    if own:
        _plan(s)
    return s


def _index(case, lengths, dev):
    """Index tensors of the packed layout: where each sequence begins and ends."""
    if case["op"] == "norm":
        return {}
    n = torch.tensor(lengths, device=dev)
    seq = torch.repeat_interleave(torch.arange(len(lengths), device=dev), n)
    end = torch.cumsum(n, 0)
    full = torch.nonzero(n).flatten()
    out = dict(seq=seq, full=full, empty=torch.nonzero(n == 0).flatten(), first=(end - n)[full], last=end[full] - 1)
    if case["op"] == "conv":
        # every sequence with its taps - 1 rows of history in front
        back = case["taps"] - 1
        row = torch.arange(sum(lengths), device=dev) + (seq + 1) * back
        ends = end + (torch.arange(len(lengths), device=dev) + 1) * back
        out.update(row=row, rows=sum(lengths) + len(lengths) * back,
                   head=((ends - n - back)[:, None] + torch.arange(back, device=dev)),
                   tail=((ends - back)[:, None] + torch.arange(back, device=dev)),
                   window=row[:, None] - back + torch.arange(back + 1, device=dev))
    return out


# ---- plain forms -----------------------------------------------------------------------------


def run(s):
    if own:
        for plan in s["plans"]:
            plan.enqueue()
        return s["out"]
    return {"conv": _plain_conv, "scan": _plain_scan, "norm": _plain_norm}[s["case"]["op"]](s)


def _silu(v):
    return v / (1 + torch.exp(-v))


def _dsilu(v):
    sg = 1 / (1 + torch.exp(-v))
    return sg * (1 + v * (1 - sg))


def _plain_conv(s):
    case, x, w = s["case"], s["x"].float(), s["w"]
    ext = x.new_zeros(s["rows"], x.shape[1])
    ext[s["row"]] = x
    if case["carry"]:
        ext[s["head"]] = s["state"].float()
    taps = ext[s["window"]]
    pre = (taps * w.t()).sum(1) + s["bias"]
    y = _silu(pre) if case["silu"] else pre
    out = {"y": y.to(s["x"].dtype)}
    if case["carry"]:
        out["new_state"] = ext[s["tail"]].to(s["x"].dtype)
    if case["train"]:
        back = case["taps"] - 1
        dpre = s["dy"].float() * _dsilu(pre) if case["silu"] else s["dy"].float()
        # dpre with zeros where a sequence has no rows, and taps - 1 more behind the last one
        wide = x.new_zeros(s["rows"] + back, x.shape[1])
        wide[s["row"]] = dpre
        ahead = torch.arange(s["rows"], device=x.device)[:, None] + torch.arange(back, -1, -1, device=x.device)
        dext = (wide[ahead] * w.t()).sum(1)
        if case["carry"]:
            dext[s["tail"]] += s["dnew_state"].float()
            out["dstate"] = dext[s["head"]].to(s["x"].dtype)
        out.update(dx=dext[s["row"]].to(s["x"].dtype), dw=(dpre[:, None, :] * taps).sum(0).t().contiguous(),
                   dbias=dpre.sum(0))
    if case["carry"] and not case["train"]:
        s["state"].copy_(out["new_state"])
        out["new_state"] = s["state"]
    return out


def _along(a, b):
    """h[t] = a[t] h[t-1] + b[t] along the first axis, by doubling."""
    step = 1
    while step < a.shape[0]:
        b = torch.cat([b[:step], b[step:] + a[step:] * b[:-step]])
        a = torch.cat([a[:step], a[step:] * a[:-step]])
        step *= 2
    return b


def _plain_scan(s):
    case, x, A, D = s["case"], s["x"].float(), s["A"], s["D"]
    total, chan = x.shape
    n, groups = case["states"], case["groups"]

    def heads(v):  # (tokens, groups * n) -> (tokens, channels, n)
        return v.float().view(total, groups, 1, n).expand(total, groups, chan // groups, n).reshape(total, chan, n)

    raw = s["dt"].float() + s["dt_bias"]
    dt = torch.where(raw > 20, raw, torch.log1p(torch.exp(torch.clamp(raw, max=20.0))))
    a = torch.exp(dt[:, :, None] * A)
    b = (dt * x)[:, :, None] * heads(s["B"])
    first, last, full, empty = s["first"], s["last"], s["full"], s["empty"]
    state = s["state"] if case["carry"] else x.new_zeros(len(s["lengths"]), chan, n)
    b[first] += a[first] * state[full]
    cut = a.clone()
    cut[first] = 0  # no state passes from one sequence to the next
    h = _along(cut, b)
    pre = (h * heads(s["C"])).sum(-1) + D * x
    z = s["z"].float() if case["gate"] else None
    out = {"y": (pre * _silu(z) if case["gate"] else pre).to(s["x"].dtype)}
    if case["carry"]:
        new = state.clone()
        new[full] = h[last]
        out["new_state"] = new
    if case["train"]:
        dy = s["dy"].float()
        dp = dy * _silu(z) if case["gate"] else dy
        grow = dp[:, :, None] * heads(s["C"])
        if case["carry"]:
            grow[last] += s["dnew_state"][full]
        after = torch.cat([cut[1:], torch.zeros_like(cut[:1])])
        g = _along(after.flip(0), grow.flip(0)).flip(0)
        prev = torch.cat([torch.zeros_like(h[:1]), h[:-1]])
        prev[first] = state[full]
        q = g * a * prev
        u = (g * heads(s["B"])).sum(-1)
        dstep = (q * A).sum(-1) + x * u
        draw_ = dstep / (1 + torch.exp(-raw))

        def joined(v):  # sum over the channels of a group
            return v.view(total, groups, chan // groups, n).sum(2).reshape(total, groups * n).to(s["x"].dtype)

        out.update(dx=(D * dp + dt * u).to(s["x"].dtype), ddt=draw_.to(s["x"].dtype),
                   dA=(q * dt[:, :, None]).sum(0), dB=joined(g * (dt * x)[:, :, None]),
                   dC=joined(dp[:, :, None] * h), dD=(dp * x).sum(0), ddt_bias=draw_.sum(0))
        if case["gate"]:
            out["dz"] = (dy * pre * _dsilu(z)).to(s["x"].dtype)
        if case["carry"]:
            dstate = s["dnew_state"].clone()
            dstate[full] = a[first] * g[first]
            out["dstate"] = dstate
    elif case["carry"]:
        s["state"].copy_(out["new_state"])
        out["new_state"] = s["state"]
    return out


def _plain_norm(s):
    case, x = s["case"], s["x"].float()
    total, chan = x.shape
    gate = s["gate"].float() if case["gate"] != "none" else None
    scale, weight, norm_weight = s["scale"], s["weight"], s["norm_weight"]
    lead = (total, case["groups"], chan // case["groups"])
    u = x * _silu(gate) if case["gate"] == "first" else x
    inv = torch.rsqrt((u.view(lead) ** 2).mean(-1, keepdim=True) + _EPS)
    hat = (u.view(lead) * inv).view(total, chan)
    v = hat * weight
    last = v * _silu(gate) if case["gate"] == "last" else v
    r = s["residual"].float() + scale * last
    rinv = torch.rsqrt((r ** 2).mean(-1, keepdim=True) + _EPS)
    out = {"y": r.to(s["x"].dtype), "h": (r * rinv * norm_weight).to(s["x"].dtype)}
    if case["train"]:
        dh = s["dh"].float()
        rhat, e = r * rinv, dh * norm_weight
        dr = s["dy"].float() + rinv * (e - rhat * (e * rhat).mean(-1, keepdim=True))
        dlast = dr * scale
        dv = dlast * _silu(gate) if case["gate"] == "last" else dlast
        dhat = (dv * weight).view(lead)
        hat3 = hat.view(lead)
        du = (inv * (dhat - hat3 * (dhat * hat3).mean(-1, keepdim=True))).view(total, chan)
        dx = du * _silu(gate) if case["gate"] == "first" else du
        out.update(dx=dx.to(s["x"].dtype), dresidual=dr.to(s["x"].dtype), dweight=(dv * hat).sum(0),
                   dscale=(dr * last).sum(0), dnorm_weight=(dh * rhat).sum(0))
        if gate is not None:
            out["dgate"] = ((du * x if case["gate"] == "first" else dlast * v) * _dsilu(gate)).to(s["x"].dtype)
    return out


# ---- the framework's plans -------------------------------------------------------------------


def _plan(s):
    """The plans that a program keeps for these buffers, on torch's current stream."""
    import numpy as np

    from nengo_ocl_b200 import cura_sequence as seq
    from nengo_ocl_b200.curaggedarray import CUDARaggedArray
    from nengo_ocl_b200.runtime import CommandQueue, DeviceArray, bfloat16

    kinds = {torch.float32: np.float32, torch.float16: np.float16, torch.bfloat16: bfloat16}
    queue = CommandQueue(stream=torch.cuda.current_stream().cuda_stream)
    case, lengths, out = s["case"], s["lengths"], {}

    def array(t):
        return DeviceArray(queue, t.shape, kinds[t.dtype], data=t.data_ptr(), base=t)

    def rows(t):  # one item per sequence of a packed (tokens, columns) tensor
        n = np.asarray(lengths)
        cols = np.full(len(n), t.shape[1])
        return CUDARaggedArray.from_buffer(queue, array(t), (np.cumsum(n) - n) * t.shape[1], n, cols, cols,
                                           np.ones(len(n), int))

    def items(t):  # one item per leading index
        k, m, n = t.shape
        return CUDARaggedArray.from_buffer(queue, array(t), np.arange(k) * m * n, np.full(k, m), np.full(k, n),
                                           np.full(k, n), np.ones(k, int))

    def new(name, like, dtype=None):
        out[name] = torch.empty_like(like, dtype=dtype)
        return out[name]

    x = s["x"]
    carry, train = case.get("carry"), case["train"]
    if carry:
        state = items(s["state"])
        out["new_state"] = torch.empty_like(s["state"]) if train else s["state"]
        new_state = items(out["new_state"]) if train else state
    if case["op"] == "conv":
        fwd = seq.plan_causal_conv(queue, rows(x), array(s["w"]), rows(new("y", x)), bias=array(s["bias"]),
                                   state=state if carry else None, new_state=new_state if carry else None,
                                   activation="silu" if case["silu"] else None)
        plans = [fwd]
        if train:
            more = dict(dstate=items(new("dstate", s["state"])), dnew_state=items(s["dnew_state"])) if carry else {}
            plans.append(seq.plan_causal_conv_grad(queue, fwd, rows(s["dy"]), rows(new("dx", x)),
                                                   array(new("dw", s["w"])), dbias=array(new("dbias", s["bias"])),
                                                   **more))
    elif case["op"] == "scan":
        fwd = seq.plan_selective_scan(
            queue, rows(x), rows(s["dt"]), array(s["A"]), rows(s["B"]), rows(s["C"]), rows(new("y", x)),
            D=array(s["D"]), Z=rows(s["z"]) if case["gate"] else None, dt_bias=array(s["dt_bias"]), softplus=True,
            state=state if carry else None, new_state=new_state if carry else None, keep=train)
        plans = [fwd]
        if train:
            more = dict(dstate=items(new("dstate", s["state"])), dnew_state=items(s["dnew_state"])) if carry else {}
            if case["gate"]:
                more["dZ"] = rows(new("dz", x))
            plans.append(seq.plan_selective_scan_grad(
                queue, fwd, rows(s["dy"]), rows(new("dx", x)), rows(new("ddt", x)), array(new("dA", s["A"])),
                rows(new("dB", s["B"])), rows(new("dC", s["C"])), dD=array(new("dD", s["D"])),
                ddt_bias=array(new("ddt_bias", s["dt_bias"])), **more))
    else:
        gated = case["gate"] != "none"
        fwd = seq.plan_residual_norm(
            queue, rows(x), Y=rows(new("y", x)), H=rows(new("h", x)), gate=rows(s["gate"]) if gated else None,
            gate_first=case["gate"] != "last", residual=rows(s["residual"]), weight=array(s["weight"]),
            scale=array(s["scale"]), norm_weight=array(s["norm_weight"]), groups=case["groups"], eps=_EPS)
        plans = [fwd]
        if train:
            plans.append(seq.plan_residual_norm_grad(
                queue, fwd, rows(new("dx", x)), dY=rows(s["dy"]), dH=rows(s["dh"]),
                dgate=rows(new("dgate", x)) if gated else None, dresidual=rows(new("dresidual", x)),
                dweight=array(new("dweight", s["weight"])), dscale=array(new("dscale", s["scale"])),
                dnorm_weight=array(new("dnorm_weight", s["norm_weight"]))))
    s.update(plans=plans, out=out)


# ---- work ------------------------------------------------------------------------------------


def work(case):
    lengths, chan = _lengths(case), case["channels"]
    total, n_seq, e = sum(lengths), len(lengths), _TYPES[case["dtype"]].itemsize
    train = case["train"]
    if case["op"] == "conv":
        taps = case["taps"]
        state = n_seq * (taps - 1) * chan * e if case["carry"] else 0
        # x in, y out, (training: x and dy in, dx out again); taps multiply-adds a value and direction
        moved = 2 * total * chan * e + 2 * state + 4 * chan * (taps + 1)
        flops = total * chan * (2 * taps + 6)
        if train:
            moved += 2 * total * chan * e + 2 * state + 4 * chan * (taps + 1)
            flops += total * chan * (4 * taps + 10)
    elif case["op"] == "scan":
        n, groups = case["states"], case["groups"]
        state = n_seq * chan * n * 4 if case["carry"] else 0
        wide = 4 if case["gate"] else 3
        moved = total * (wide * chan + 2 * groups * n) * e + 2 * state + 4 * chan * (n + 2)
        flops = total * chan * (7 * n + 20)
        if train:  # dy in, the gradients out
            moved += total * (wide * chan + 2 * groups * n) * e + 2 * state + 4 * chan * (n + 2)
            flops += total * chan * (19 * n + 30)
    else:
        wide = 4 if case["gate"] == "none" else 5
        moved = total * wide * chan * e + 12 * chan
        flops = total * chan * 16
        if train:  # dy and dh in, the gradients of x, of the gate and of the residual out
            moved += total * wide * chan * e + 12 * chan
            flops += total * chan * 40
    return {"bytes": moved, "flops": flops}


# ---- definitions in 64 bits ------------------------------------------------------------------


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    fields = ("x", "w", "bias", "state", "dt", "dt_bias", "A", "B", "C", "D", "z", "residual", "weight", "norm_weight",
              "scale", "gate")
    leaf = {k: s[k].double().requires_grad_(case["train"]) for k in fields if isinstance(s.get(k), torch.Tensor)}
    make = {"conv": _exact_conv, "scan": _exact_scan, "norm": _exact_norm}[case["op"]]
    out, pairs = make(case, s, leaf)
    if not case["train"]:
        return out
    heads = [out[k] for k in pairs]
    keys = list(leaf)
    grads = torch.autograd.grad(heads, [leaf[k] for k in keys], [s[g].double().reshape(out[k].shape)
                                                                 for k, g in pairs.items()], allow_unused=True)
    out = {k: v.detach() for k, v in out.items()}
    for k, g in zip(keys, grads):
        out["d" + k] = torch.zeros_like(leaf[k]) if g is None else g
    return out


def _exact_conv(case, s, v):
    ys, ends = [], []
    begin, back = 0, case["taps"] - 1
    for k, n in enumerate(s["lengths"]):
        before = v["state"][k] if case["carry"] else v["x"].new_zeros(back, v["x"].shape[1])
        line = torch.cat([before, v["x"][begin:begin + n]])
        begin += n
        pre = v["bias"].expand(n, -1)
        for j in range(back + 1):
            pre = pre + v["w"][:, j] * line[j:j + n]
        ys.append(pre * torch.sigmoid(pre) if case["silu"] else pre)
        ends.append(line[n:])
    out = {"y": torch.cat(ys)}
    pairs = {"y": "dy"}
    if case["carry"]:
        out["new_state"] = torch.stack(ends)
        pairs["new_state"] = "dnew_state"
    return out, pairs


def _exact_scan(case, s, v):
    chan, n = v["A"].shape
    of = torch.arange(chan, device=v["A"].device) // (chan // case["groups"])
    ys, ends, begin = [], [], 0
    step = torch.nn.functional.softplus(v["dt"] + v["dt_bias"], threshold=50.0)
    line = [w.unbind(0) for w in (step, step * v["x"], v["B"], v["C"])]
    for k, length in enumerate(s["lengths"]):
        h = v["state"][k] if case["carry"] else v["A"].new_zeros(chan, n)
        for t in range(begin, begin + length):
            d, dx, b, c = (w[t] for w in line)
            h = torch.exp(d[:, None] * v["A"]) * h + dx[:, None] * b.view(-1, n)[of]
            ys.append((h * c.view(-1, n)[of]).sum(1))
        begin += length
        ends.append(h)
    y = torch.stack(ys) + v["D"] * v["x"]
    out = {"y": y * v["z"] * torch.sigmoid(v["z"]) if case["gate"] else y}
    pairs = {"y": "dy"}
    if case["carry"]:
        out["new_state"] = torch.stack(ends)
        pairs["new_state"] = "dnew_state"
    return out, pairs


def _exact_norm(case, s, v):
    def unit(u):
        return u / torch.sqrt(u.square().mean(-1, keepdim=True) + _EPS)

    u = v["x"]
    if case["gate"] == "first":
        u = u * v["gate"] * torch.sigmoid(v["gate"])
    u = unit(u.unflatten(1, (case["groups"], -1))).flatten(1) * v["weight"]
    if case["gate"] == "last":
        u = u * v["gate"] * torch.sigmoid(v["gate"])
    r = v["residual"] + v["scale"] * u
    return {"y": r, "h": unit(r) * v["norm_weight"]}, {"y": "dy", "h": "dh"}
