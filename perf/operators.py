"""What is measured of the multi-axis rotary positions and of differential attention.

Rotary positions.  Token r carries A integer coordinates pos[r, a] (time,
height, width); axis a owns pairs[a] pairs of each head's columns, pair p turns
by the angle pos[r, axis(p)] * inv_freq[p].  The backward pass is the inverse
rotation of the gradient.

Differential attention.  A head's queries and keys are 2*dh wide, two halves
of dh; its values are 2*dh wide.  With s_m = scale * q_m k_m^T over the visible
keys and P_m = softmax(s_m), the output is (P_1 - lam * P_2) v, lam one learned
weight per head.  A query that sees no key has output 0 and no gradient.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def listed():
    return [
        # the q and k of one decoded token per sequence: latency only
        {"name": "rope_token_bf16", "op": "rope", "type": "bf16", "rows": 8, "heads": 24, "dh": 64, "axes": 1,
         "part": 0, "inter": False, "back": False},
        # 8x8 image tokens of a batch of 128, width 256: q and k of the fused projection
        {"name": "rope_image_f32", "op": "rope", "type": "f32", "rows": 128 * 64, "heads": 16, "dh": 32, "axes": 2,
         "part": 0, "inter": False, "back": False},
        # gradient of q and k for packed images of odd sizes, adjacent pairs, a quarter of the columns unrotated
        {"name": "rope_packed_back_f32", "op": "rope", "type": "f32", "rows": 30011, "heads": 12, "dh": 48, "axes": 2,
         "part": 6, "inter": True, "back": True},
        # two clips of 16 frames of 32x32 tokens, q and k of 16 heads
        {"name": "rope_video_bf16", "op": "rope", "type": "bf16", "rows": 2 * 16 * 1024, "heads": 32, "dh": 64,
         "axes": 3, "part": 0, "inter": False, "back": False},
        # one new token against a short cache in f32: latency only
        {"name": "diff_token_short_f32", "op": "diff", "type": "f32", "n": 2, "h": 4, "hkv": 4, "dh": 32, "tq": 1,
         "tk": 777, "causal": "end", "ragged": True, "mask": False, "train": False},
        # one new token for 8 sequences over caches of up to 32768 keys, four query heads to a key head
        {"name": "diff_token_long_bf16", "op": "diff", "type": "bf16", "n": 8, "h": 16, "hkv": 4, "dh": 64, "tq": 1,
         "tk": 32768, "causal": "end", "ragged": True, "mask": False, "train": False},
        # a batch of 128 images of 8x8 tokens in f32, four heads of 64 columns: forward for evaluation
        {"name": "diff_image_f32", "op": "diff", "type": "f32", "n": 128, "h": 4, "hkv": 4, "dh": 32, "tq": 64,
         "tk": 64, "causal": "", "ragged": False, "mask": False, "train": False},
        # training on 16x16 tokens in f32, dropped patches masked out
        {"name": "diff_image_train_f32", "op": "diff", "type": "f32", "n": 32, "h": 4, "hkv": 4, "dh": 32, "tq": 256,
         "tk": 256, "causal": "", "ragged": False, "mask": True, "train": True},
        # ragged training batch of odd lengths with shared key heads, narrow heads; some sequences may be empty
        {"name": "diff_ragged_train_bf16", "op": "diff", "type": "bf16", "n": 5, "h": 6, "hkv": 2, "dh": 40,
         "tq": 1003, "tk": 1003, "causal": "start", "ragged": True, "mask": False, "train": True},
        # cross attention from 8x8 queries to a 16x16 memory, trained in bf16
        {"name": "diff_cross_train_bf16", "op": "diff", "type": "bf16", "n": 128, "h": 6, "hkv": 6, "dh": 32,
         "tq": 64, "tk": 256, "causal": "", "ragged": False, "mask": False, "train": True},
        # a prompt or clip of 8192 tokens read at once
        {"name": "diff_long_bf16", "op": "diff", "type": "bf16", "n": 2, "h": 8, "hkv": 4, "dh": 64, "tq": 8192,
         "tk": 8192, "causal": "start", "ragged": False, "mask": False, "train": False},
        # training over all tokens of a clip of 8 frames of 32x32
        {"name": "diff_clip_train_bf16", "op": "diff", "type": "bf16", "n": 1, "h": 8, "hkv": 8, "dh": 64,
         "tq": 8192, "tk": 8192, "causal": "", "ragged": False, "mask": False, "train": True},
    ]


def _spread(rng, low, high):
    """A whole number between low and high, even over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["rope", "token", "fwd", "train", "train"])
    typ = rng.choice(["f32", "bf16", "bf16"])
    if kind == "rope":
        heads, axes, dh = rng.randint(1, 48), rng.randint(1, 4), 4 * rng.randint(4, 32)
        rows = _spread(rng, 1, min(60000, 60_000_000 // (heads * dh)))
        return {"op": "rope", "type": typ, "rows": rows, "heads": heads, "dh": dh, "axes": axes,
                "part": rng.choice([0, 0, 2]), "inter": rng.random() < 0.4, "back": rng.random() < 0.4}
    hkv = rng.choice([1, 2, 3, 4, 8])
    h = hkv * rng.choice([1, 1, 2, 4])
    dh = rng.choice([8, 16, 24, 32, 32, 40, 64, 64, 64])
    ragged, mask = rng.random() < 0.5, rng.random() < 0.3
    if kind == "token":
        tk = _spread(rng, 64, 60000)
        n = _spread(rng, 1, max(1, min(64, 1_000_000 // (tk * hkv))))
        tq = rng.choice([1, 1, 1, 2, 5])
        return {"op": "diff", "type": typ, "n": n, "h": h, "hkv": hkv, "dh": dh, "tq": tq, "tk": tk, "causal": "end",
                "ragged": ragged, "mask": mask, "train": False}
    room = (1 << 28) if typ == "bf16" else (1 << 25)
    top = 8192 if typ == "bf16" else 2500
    tq = _spread(rng, 16, min(top, math.isqrt(room // h)))
    tk = tq if rng.random() < 0.6 else _spread(rng, 16, min(top, room // (tq * h)))
    n = _spread(rng, 1, max(1, min(128, room // (tq * tk * h))))
    causal = rng.choice(["", "start", "end"]) if tq == tk else rng.choice(["", "end"])
    return {"op": "diff", "type": typ, "n": n, "h": h, "hkv": hkv, "dh": dh, "tq": tq, "tk": tk, "causal": causal,
            "ragged": ragged, "mask": mask, "train": kind == "train"}


def _pairs(case):
    """The pairs of each axis: `part` pairs stay unrotated, the others are shared out, the first axes one more."""
    total, a = case["dh"] // 2 - case["part"], case["axes"]
    return tuple(total // a + (1 if i < total % a else 0) for i in range(a))


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    typ, dev = TYPES[case["type"]], "cuda"

    def normal(*shape):
        return torch.randn(*shape, device=dev, generator=g).to(typ)

    if case["op"] == "rope":
        pairs = _pairs(case)
        freq = [10000.0 ** (-j / max(1, p)) for p in pairs for j in range(p)]
        pos = torch.randint(0, 200, (case["rows"], case["axes"]), device=dev, generator=g, dtype=torch.int32)
        return {"case": dict(case), "x": normal(case["rows"], case["heads"], case["dh"]), "pos": pos, "pairs": pairs,
                "freq": torch.tensor(freq, dtype=torch.float32, device=dev)}
    n, h, hkv, w, tq, tk = (case[k] for k in ("n", "h", "hkv", "dh", "tq", "tk"))
    w *= 2
    s = {"case": dict(case), "scale": (w // 2) ** -0.5, "klen": None, "mask": None}
    if tq == tk and h == hkv:  # one projection's output, as a self-attention layer has it
        qkv = normal(n, tq, 3, h, w)
        s["q"], s["k"], s["v"] = qkv[:, :, 0], qkv[:, :, 1], qkv[:, :, 2]
    else:
        s["q"], kv = normal(n, tq, h, w), normal(n, tk, 2, hkv, w)
        s["k"], s["v"] = kv[:, :, 0], kv[:, :, 1]
    s["lam"] = 0.2 + 0.6 * torch.rand(h, device=dev, generator=g)
    if case["ragged"]:
        low = 0 if case["train"] else tk // 2
        s["klen"] = torch.randint(low, tk + 1, (n,), device=dev, generator=g, dtype=torch.int32)
        s["klen"][0] = tk
    if case["mask"]:
        s["mask"] = torch.rand(n, tk, device=dev, generator=g) < 0.75
    if case["train"]:
        s["dout"] = normal(n, tq, h, w)
    return s


def run(state):
    case = state["case"]
    if case["op"] == "rope":
        return _rope_own(state) if own else _rope_plain(state)
    return _diff_own(state) if own else _diff_plain(state)


def _rope_own(s):
    from rustnn_b200 import ops

    f = ops.rope_backward if s["case"]["back"] else ops.rope
    return f(s["x"], s["pos"], s["freq"], s["pairs"], interleaved=s["case"]["inter"])


def _rope_plain(s):
    case, pairs = s["case"], s["pairs"]
    x, total = s["x"].float(), sum(s["pairs"])
    axis = torch.repeat_interleave(torch.arange(len(pairs), device=x.device),
                                   torch.tensor(pairs, device=x.device), output_size=total)
    angle = s["pos"].float()[:, axis] * s["freq"]
    c, d = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
    if case["back"]:
        d = -d
    rot, rest = x[..., : 2 * total], x[..., 2 * total:]
    if case["inter"]:
        a, b = rot[..., 0::2], rot[..., 1::2]
        y = torch.stack([a * c - b * d, a * d + b * c], -1).flatten(-2)
    else:
        a, b = rot[..., :total], rot[..., total:]
        y = torch.cat([a * c - b * d, a * d + b * c], -1)
    return torch.cat([y, rest], -1).to(s["x"].dtype)


def _diff_own(s):
    from rustnn_b200 import ops

    case = s["case"]
    how = {"scale": s["scale"], "causal": case["causal"] or None, "klen": s["klen"], "kmask": s["mask"]}
    if not case["train"]:
        return ops.diffattn_forward(s["q"], s["k"], s["v"], s["lam"], **how)
    o, o2, lse = ops.diffattn_forward(s["q"], s["k"], s["v"], s["lam"], save=True, **how)
    dlam = torch.zeros_like(s["lam"])
    dq, dk, dv = ops.diffattn_backward(s["dout"], s["q"], s["k"], s["v"], s["lam"], o, o2, lse, dlam, **how)
    return {"o": o, "dq": dq, "dk": dk, "dv": dv, "dlam": dlam}


def _visible(s):
    """[n, 1, 1, tq, tk]: whether query i sees key j."""
    case = s["case"]
    n, tq, tk = case["n"], case["tq"], case["tk"]
    dev = s["q"].device
    i, j = torch.arange(tq, device=dev)[:, None], torch.arange(tk, device=dev)[None]
    length = s["klen"][:, None, None] if s["klen"] is not None else torch.full((n, 1, 1), tk, device=dev)
    see = (j < length).expand(n, tq, tk)
    if case["causal"] == "start":
        see = see & (j <= i)
    elif case["causal"] == "end":
        see = see & (j <= i + length - tq)
    if s["mask"] is not None:
        see = see & s["mask"][:, None]
    return see[:, None, None]


def _diff_plain(s):
    case = s["case"]
    n, h, hkv, dh, tq, tk = (case[k] for k in ("n", "h", "hkv", "dh", "tq", "tk"))
    grp, typ = h // hkv, s["q"].dtype
    # [n, hkv, grp, t, columns]; the keys and values of a group broadcast over its query heads
    q = s["q"].float().reshape(n, tq, hkv, grp, 2 * dh).permute(0, 2, 3, 1, 4)
    k = s["k"].float().permute(0, 2, 1, 3)[:, :, None]
    v = s["v"].float().permute(0, 2, 1, 3)[:, :, None]
    lam = s["lam"].view(1, hkv, grp, 1, 1)
    hide = ~_visible(s)

    def softmax(a, b):
        w = (a @ b.transpose(-1, -2) * s["scale"]).masked_fill_(hide, -math.inf)
        top = w.amax(-1, keepdim=True)
        w = w.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)).exp_()
        total = w.sum(-1, keepdim=True)
        return w.div_(torch.where(total == 0, torch.ones_like(total), total))

    def heads_last(x):
        return x.permute(0, 3, 1, 2, 4).reshape(n, x.shape[3], -1, 2 * dh).to(typ)

    p1, p2 = softmax(q[..., :dh], k[..., :dh]), softmax(q[..., dh:], k[..., dh:])
    o = heads_last((p1 - lam * p2) @ v)
    if not case["train"]:
        return o
    do = s["dout"].float().reshape(n, tq, hkv, grp, 2 * dh).permute(0, 2, 3, 1, 4)
    dv = ((p1 - lam * p2).transpose(-1, -2) @ do).sum(2, keepdim=True)
    dp = do @ v.transpose(-1, -2)
    r1, r2 = (p1 * dp).sum(-1, keepdim=True), (p2 * dp).sum(-1, keepdim=True)
    ds1 = (dp - r1).mul_(p1).mul_(s["scale"])
    ds2 = dp.sub_(r2).mul_(p2).mul_(-s["scale"] * lam)
    dq = torch.cat([ds1 @ k[..., :dh], ds2 @ k[..., dh:]], -1)
    dk = torch.cat([ds1.transpose(-1, -2) @ q[..., :dh], ds2.transpose(-1, -2) @ q[..., dh:]], -1)
    return {"o": o, "dq": heads_last(dq), "dk": heads_last(dk.sum(2, keepdim=True)), "dv": heads_last(dv),
            "dlam": -r2.sum((0, 3, 4)).reshape(h)}


def _seen(case):
    """How many (query, key) pairs of one head and sequence the path has to look at."""
    tq, tk = case["tq"], case["tk"]
    if not case["causal"]:
        return tq * tk
    first = 1 if case["causal"] == "start" else tk - tq + 1  # keys that query 0 sees
    return sum(min(tk, max(0, first + i)) for i in range(tq))


def work(case):
    size = 4 if case["type"] == "f32" else 2
    if case["op"] == "rope":
        total = case["rows"] * case["heads"] * case["dh"]
        return {"bytes": 2 * total * size + case["rows"] * case["axes"] * 4, "flops": 3 * total}
    n, h, hkv, dh, tq, tk = (case[k] for k in ("n", "h", "hkv", "dh", "tq", "tk"))
    share = (0.5 if case["train"] else 0.75) if case["ragged"] and n > 1 else 1.0
    rows, keys = n * h * tq * 2 * dh * size, 2 * n * hkv * tk * 2 * dh * size * share
    # a pair costs two products of dh columns for the scores and one of 2*dh for the combined map;
    # the gradient costs the scores again, dP and dV of 2*dh, dQ and dK of 2*dh
    flops = 2.0 * n * h * _seen(case) * share * 4 * dh
    if not case["train"]:
        return {"bytes": 2 * rows + keys, "flops": flops}
    return {"bytes": 4 * rows + 2 * keys, "flops": 3.5 * flops}


def exact(case, seed):
    s = prepare(case, seed)
    return _rope_exact(s) if case["op"] == "rope" else _diff_exact(s)


def _rope_exact(s):
    """Each pair as a complex number times exp(i * angle)."""
    case, x = s["case"], s["x"].double()
    sign = -1.0 if case["back"] else 1.0
    out, at, total = x.clone(), 0, sum(s["pairs"])
    for a, count in enumerate(s["pairs"]):
        for _ in range(count):
            turn = torch.polar(torch.ones(case["rows"], dtype=torch.float64, device=x.device),
                               sign * s["pos"][:, a].double() * s["freq"][at].double())
            i, j = (2 * at, 2 * at + 1) if case["inter"] else (at, at + total)
            z = torch.complex(x[..., i], x[..., j]) * turn[:, None]
            out[..., i], out[..., j] = z.real, z.imag
            at += 1
    return out


def _diff_exact(s):
    """Head by head and sequence by sequence from the definition, the gradient by autograd in 64 bits."""
    case = s["case"]
    n, h, hkv, dh, tq, tk = (case[k] for k in ("n", "h", "hkv", "dh", "tq", "tk"))
    if n * h * tq * tk > 1.2e9:
        return None
    q, k, v = (s[x].double().requires_grad_(case["train"]) for x in ("q", "k", "v"))
    lam = s["lam"].double().requires_grad_(case["train"])
    see = _visible(s)[:, 0, 0]
    o = torch.zeros(n, tq, h, 2 * dh, dtype=torch.float64, device=q.device)
    for b in range(n):
        some = see[b].any(-1, keepdim=True)
        bias = torch.zeros(tq, tk, dtype=torch.float64, device=q.device).masked_fill(~see[b] & some, -math.inf)
        for e in range(h):
            f = e // (h // hkv)
            maps = [torch.softmax(q[b, :, e, c] @ k[b, :, f, c].T * s["scale"] + bias, -1)
                    for c in (slice(0, dh), slice(dh, 2 * dh))]
            one = ((maps[0] - lam[e] * maps[1]) @ v[b, :, f]) * some
            o[b, :, e] = one.detach()
            if case["train"]:
                one.backward(s["dout"][b, :, e].double())
    if not case["train"]:
        return o
    return {"o": o, "dq": q.grad, "dk": k.grad, "dv": v.grad, "dlam": lam.grad}
