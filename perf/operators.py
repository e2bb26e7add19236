"""The packed-row operators -- attention over documents, rotary positions, group norm with an activation -- as measured cases.

A batch of ragged utterances is a table of rows (M, ...) in which document b owns the rows [offset[b], offset[b + 1]) (``docs``
documents, the rows behind the last offset belong to nobody), or a padded cache in which document b owns the first ``length[b]`` of
``longest`` rows.  ``run`` computes one operator on such a table: with ``own`` false in its plain form (elementary torch operations in 32
bits, rounded once at the end), with ``own`` true through ``optispeech_amd.packed_ops``.

Formulas (query i of a document has the position  pos_i = keys - queries + i  among that document's keys, key j the position j):

  attention   x = scale q_i . k_j;  c = cap tanh(x / cap)  (cap > 0);  s = c - slope_h |pos_i - j|
              seen(i, j): same document, and  full: always;  causal: j <= pos_i;  prefix: j <= pos_i or j < prefix_b
              o_i = sum_j softmax_j(s over the seen keys) v_j,  0 where nothing is seen;  query head h reads key head h // (heads / shared)
  rotary      angle = (first_b + row in document) f_i;  (a, b) -> mag (a cos - b sin, a sin + b cos) over the pairs of the first ``turned``
              channels, interleaved (2 i, 2 i + 1) or half (i, i + turned / 2);  the remaining channels pass
              f_i = base^(-2 i / turned), for long contexts divided by a factor (linear), with a larger base (base), or divided only
              where a frequency makes few turns within the original length (parts; then mag = 1 + 0.1 ln factor)
  group norm  mean and variance over a document's rows and a group's channels;  y = act(w (x - mean) / sqrt(var + eps) + b)
"""
import math
import random

import torch

own = False

BASE = 10000.0
ORIGINAL = 2000                      # rows the unscaled rotary frequencies were made for (the text embedding's max_source_positions)
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


# ------------------------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one new frame for each of eight streams over a short cache, two heads of 128 as in the Transformer backbone: latency
        dict(name="token_short", op="attention", dir="token", type="bf16", docs=8, shortest=40, longest=800, mix=1, tail=0,
             heads=2, shared=2, width=128, mask="causal", cap=0.0, slope=False),
        # one new token for each of 48 requests over long caches with shared key heads and capped scores: the cache's bandwidth
        dict(name="token_long", op="attention", dir="token", type="bf16", docs=48, shortest=1, longest=16384, mix=2, tail=0,
             heads=16, shared=2, width=128, mask="causal", cap=30.0, slope=False),
        # ragged prompts packed behind each other, distances penalised per head, forward only
        dict(name="prompts", op="attention", dir="forward", type="bf16", docs=24, shortest=1, longest=2048, mix=3, tail=37,
             heads=8, shared=8, width=64, mask="causal", cap=0.0, slope=True),
        # the decoder's training batch: 32 utterances of up to 800 frames, every frame sees its whole utterance
        dict(name="utterances", op="attention", dir="train", type="bf16", docs=32, shortest=600, longest=800, mix=4, tail=0,
             heads=2, shared=2, width=128, mask="full", cap=0.0, slope=True),
        # the same in exact 32-bit arithmetic at a smaller batch, with a bidirectional prompt, caps and shared heads
        dict(name="utterances_f32", op="attention", dir="train", type="f32", docs=16, shortest=37, longest=401, mix=5, tail=5,
             heads=4, shared=2, width=64, mask="prefix", cap=20.0, slope=False),
        # long documents in training, shared heads, a bidirectional prefix and capped scores: the matrix pipe
        dict(name="documents", op="attention", dir="train", type="bf16", docs=5, shortest=1000, longest=8192, mix=6, tail=11,
             heads=16, shared=4, width=128, mask="prefix", cap=50.0, slope=False),
        # positions of one new token per stream, far out: latency
        dict(name="rotary_token", op="rotary", dir="forward", type="bf16", docs=8, shortest=1, longest=1, mix=7, tail=0, first=100000,
             heads=2, shared=2, width=128, turned=128, layout="half", scaling="base", factor=8.0),
        # a training step's rows, scaled for a long context
        dict(name="rotary_rows", op="rotary", dir="train", type="bf16", docs=16, shortest=500, longest=4096, mix=8, tail=3, first=0,
             heads=16, shared=4, width=128, turned=128, layout="half", scaling="parts", factor=8.0),
        # half of every head turned, interleaved pairs, 32 bits
        dict(name="rotary_part", op="rotary", dir="forward", type="f32", docs=32, shortest=300, longest=800, mix=9, tail=9, first=7,
             heads=4, shared=4, width=64, turned=32, layout="interleaved", scaling="linear", factor=4.0),
        # two short utterances: latency
        dict(name="norm_small", op="group_norm", dir="forward", type="f32", docs=2, shortest=17, longest=37, mix=10, tail=0,
             channels=64, groups=4, act="silu"),
        # the convolution module's rows of a large synthesis batch, trained in bf16
        dict(name="norm_rows", op="group_norm", dir="train", type="bf16", docs=64, shortest=386, longest=772, mix=11, tail=21,
             channels=384, groups=8, act="silu"),
        # the decoder's training batch in 32 bits
        dict(name="norm_f32", op="group_norm", dir="train", type="f32", docs=32, shortest=600, longest=800, mix=12, tail=0,
             channels=256, groups=32, act="gelu"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the same ranges; redrawn until it costs no more than the dearest listed case of its operator."""
    top = {}
    for c in listed():
        w = work(c)
        for key in ("bytes", "flops"):
            top[c["op"], key] = max(top.get((c["op"], key), 0), w[key])
    while True:
        op = rng.choice(["attention", "attention", "rotary", "group_norm"])
        case = dict(op=op, type=rng.choice(["bf16", "bf16", "f32"]), mix=rng.randrange(1 << 30))
        if op == "attention":
            shared = rng.choice([1, 2, 3, 4])
            case.update(dir=rng.choice(["token", "forward", "train"]), heads=shared * rng.choice([1, 2, 4, 8]), shared=shared,
                        width=rng.choice([32, 40, 64, 80, 96, 128]), mask=rng.choice(["full", "causal", "prefix"]),
                        cap=rng.choice([0.0, 0.0, 15.0, 30.0, 50.0]), slope=rng.random() < 0.4)
            longest = _log_int(rng, 4, 16384 if case["dir"] == "token" else 8192 if case["type"] == "bf16" else 1500)
            case.update(docs=_log_int(rng, 1, 64), longest=longest, shortest=rng.randint(1, longest))
        elif op == "rotary":
            shared, width = rng.choice([1, 2, 4]), rng.choice([32, 64, 80, 128])
            longest = _log_int(rng, 1, 4096)
            case.update(dir=rng.choice(["forward", "train"]), heads=shared * rng.choice([1, 2, 4]), shared=shared, width=width,
                        turned=rng.choice([width, width // 2]), layout=rng.choice(["half", "interleaved"]),
                        scaling=rng.choice(["none", "linear", "base", "parts"]), factor=rng.choice([2.0, 4.0, 8.0, 16.0]),
                        first=rng.choice([0, 0, _log_int(rng, 1, 1000000)]), docs=_log_int(rng, 1, 64), longest=longest,
                        shortest=rng.randint(1, longest))
        else:
            groups, longest = rng.choice([1, 2, 4, 8, 16, 32]), _log_int(rng, 4, 2000)
            # (relu has no gradient at 0, where a last bit decides: forward only)
            case.update(dir=rng.choice(["forward", "train"]), groups=groups, channels=groups * rng.choice([5, 8, 12, 16, 24, 32]))
            case.update(act=rng.choice(["none", "gelu", "silu"] + (["relu"] if case["dir"] == "forward" else [])),
                        docs=_log_int(rng, 1, 64), longest=longest, shortest=rng.randint(1, longest))
        case["tail"] = rng.choice([0, rng.randint(1, 50)])
        w = work(case)
        if all(w[key] <= top[op, key] for key in ("bytes", "flops")):
            return case


def lengths(case):
    """Rows of each document: the first document is the longest, the others lie between the two bounds."""
    r = random.Random(case["mix"])
    return [case["longest"]] + [r.randint(case["shortest"], case["longest"]) for _ in range(case["docs"] - 1)]


def prefixes(case):
    """Keys of each document that all its queries see (mask "prefix")."""
    r = random.Random(case["mix"] + 1)
    return [r.randint(0, max(1, n // 4)) for n in lengths(case)]


def work(case):
    """Bytes (each input once, each output once) and operations of one pass."""
    size, ls = (2 if case["type"] == "bf16" else 4), lengths(case)
    if case["op"] == "attention":
        pairs = 0
        for n, p in zip(ls, prefixes(case)):
            if case["dir"] == "token":
                pairs += n
            elif case["mask"] == "full":
                pairs += n * n
            else:
                p = p if case["mask"] == "prefix" else 0
                pairs += n * (n + 1) // 2 + p * (p - 1) // 2
        queries = case["docs"] if case["dir"] == "token" else sum(ls)
        qo, kv = queries * case["heads"] * case["width"] * size, sum(ls) * case["shared"] * case["width"] * size
        train = case["dir"] == "train"
        # forward: q, k, v in, o out;  training adds the incoming gradient and the three outgoing ones
        return {"bytes": (4 if train else 2) * qo + (4 if train else 2) * kv,
                "flops": (14 if train else 4) * pairs * case["heads"] * case["width"]}
    if case["op"] == "rotary":
        n = sum(ls) * (case["heads"] + case["shared"]) * case["width"]
        turned = sum(ls) * (case["heads"] + case["shared"]) * case["turned"]
        passes = 2 if case["dir"] == "train" else 1
        return {"bytes": 2 * passes * n * size, "flops": 3 * passes * turned}
    n, c = sum(ls) * case["channels"], case["channels"]
    if case["dir"] == "train":                                # x, dy in; y, dx out; weights and their gradients
        return {"bytes": 4 * n * size + 16 * c, "flops": 24 * n}
    return {"bytes": 2 * n * size + 8 * c, "flops": 8 * n}


# ------------------------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    dev, dt = torch.device("cuda"), TYPES[case["type"]]
    g = torch.Generator(device=dev).manual_seed(seed * 7919 + case["mix"] % 7919)
    ls = lengths(case)
    total = sum(ls) + case["tail"]
    offsets = [0]
    for n in ls:
        offsets.append(offsets[-1] + n)
    st = dict(case=case, lengths=ls, total=total, offsets=torch.tensor(offsets, dtype=torch.int64, device=dev))

    def randn(*shape, std=1.0, dtype=dt):
        return (torch.randn(shape, generator=g, device=dev) * std).to(dtype)

    train = case["dir"] == "train"
    if case["op"] == "attention":
        H, S, D = case["heads"], case["shared"], case["width"]
        token = case["dir"] == "token"
        queries, keys = (case["docs"], case["docs"] * case["longest"]) if token else (total, total)
        # capped scores are capped because they grow large: queries a few times the unit scale there
        st.update(q=randn(queries, H, D, std=4.0 if case["cap"] else 1.0), k=randn(keys, S, D), v=randn(keys, S, D))
        st["slopes"] = torch.tensor([2.0 ** (-8.0 * (h + 1) / H) for h in range(H)], device=dev) if case["slope"] else None
        st["prefix"] = torch.tensor(prefixes(case), dtype=torch.int64, device=dev) if case["mask"] == "prefix" else None
        st["prefixes"] = prefixes(case) if case["mask"] == "prefix" else [0] * case["docs"]
        st["scale"] = D ** -0.5
        if token:
            st["key_lengths"] = torch.tensor(ls, dtype=torch.int64, device=dev)
            st["token_offsets"] = torch.arange(case["docs"] + 1, dtype=torch.int64, device=dev)
        grads = dict(do=randn(queries, H, D)) if train else {}
        leaves = ("q", "k", "v")
    elif case["op"] == "rotary":
        st.update(q=randn(total, case["heads"], case["width"]), k=randn(total, case["shared"], case["width"]))
        r = random.Random(seed)
        st["firsts"] = [case["first"] + (r.randrange(1000) if case["first"] else 0) for _ in ls]
        st["first"] = torch.tensor(st["firsts"], dtype=torch.int64, device=dev) if case["first"] else None
        grads = dict(dq=randn(total, case["heads"], case["width"]), dk=randn(total, case["shared"], case["width"])) if train else {}
        leaves = ("q", "k")
    else:
        C = case["channels"]
        # channel offsets and scales as a convolution leaves them: the means are not small next to the deviations
        centre, spread = randn(C, std=2.0, dtype=torch.float32), randn(C, dtype=torch.float32).abs() + 0.25
        st["x"] = (torch.randn((total, C), generator=g, device=dev) * spread + centre).to(dt)
        st["w"] = torch.nn.Parameter(randn(C, std=0.2, dtype=torch.float32) + 1.0)
        st["b"] = torch.nn.Parameter(randn(C, std=0.2, dtype=torch.float32))
        st["eps"] = 1e-5
        grads = dict(dy=randn(total, C)) if train else {}
        leaves = ("x",)
    st.update(grads)
    if train:
        for name in leaves:
            st[name].requires_grad_(True)
    if own:
        from optispeech_amd import packed_ops
        if case["op"] == "attention" and case["dir"] == "token":
            st["rows"] = packed_ops.PackedRows.from_offsets(st["token_offsets"], case["docs"], longest=1)
            st["keys"] = packed_ops.PackedRows.from_padded(st["key_lengths"], case["longest"])
        else:
            st["rows"] = packed_ops.PackedRows.from_offsets(st["offsets"], total, longest=case["longest"])
            st["keys"] = None
        if case["op"] == "rotary":
            st["rope"] = packed_ops.Rotary(case["turned"], base=BASE, layout=case["layout"], scaling=case["scaling"],
                                           factor=case["factor"], original_length=ORIGINAL, device=dev)
    return st


# ------------------------------------------------------------------------------------------------------------------ one pass
def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(st):
    from optispeech_amd import packed_ops
    case = st["case"]
    train = case["dir"] == "train"
    with torch.set_grad_enabled(train):
        if case["op"] == "attention":
            o = packed_ops.attention(st["q"], st["k"], st["v"], st["rows"], keys=st["keys"], causal=case["mask"] != "full",
                                     prefix=st["prefix"], softcap=case["cap"], slopes=st["slopes"], scale=st["scale"])
            return (o,) + torch.autograd.grad(o, (st["q"], st["k"], st["v"]), st["do"]) if train else o
        if case["op"] == "rotary":
            q, k = packed_ops.rotary(st["q"], st["k"], st["rope"], st["rows"], first=st["first"])
            return (q, k) + torch.autograd.grad((q, k), (st["q"], st["k"]), (st["dq"], st["dk"])) if train else (q, k)
        y = packed_ops.group_norm(st["x"], st["w"], st["b"], case["groups"], st["rows"], eps=st["eps"], act=case["act"])
        if not train:
            return y
        st["w"].grad = st["b"].grad = None                    # parameter gradients accumulate: a step starts them anew
        (dx,) = torch.autograd.grad(y, (st["x"],), st["dy"])
        return y, dx, st["w"].grad, st["b"].grad


def _run_plain(st):
    case = st["case"]
    train = case["dir"] == "train"
    with torch.set_grad_enabled(train):
        if case["op"] == "attention":
            o = _plain_attention(st)
            return (o,) + torch.autograd.grad(o, (st["q"], st["k"], st["v"]), st["do"]) if train else o
        if case["op"] == "rotary":
            q, k = _plain_rotary(st)
            return (q, k) + torch.autograd.grad((q, k), (st["q"], st["k"]), (st["dq"], st["dk"])) if train else (q, k)
        y = _plain_group_norm(st)
        return (y,) + torch.autograd.grad(y, (st["x"], st["w"], st["b"]), st["dy"]) if train else y


def _plain_attention(st):
    case, ls = st["case"], st["lengths"]
    q, k, v, S = st["q"], st["k"], st["v"], case["shared"]
    group = case["heads"] // S
    if case["dir"] == "token":
        parts = [(q[b:b + 1], k[b * case["longest"]:b * case["longest"] + n], v[b * case["longest"]:b * case["longest"] + n])
                 for b, n in enumerate(ls)]
        tail = 0
    else:
        sizes = ls + [st["total"] - sum(ls)]
        parts = list(zip(q.split(sizes), k.split(sizes), v.split(sizes)))[:-1]
        tail = sizes[-1]
    out = []
    for b, (qd, kd, vd) in enumerate(parts):
        qf = qd.float().transpose(0, 1)                                                       # (H, queries, D)
        kf = kd.float().transpose(0, 1).repeat_interleave(group, 0)                           # (H, keys, D)
        vf = vd.float().transpose(0, 1).repeat_interleave(group, 0)
        s = torch.matmul(qf, kf.transpose(1, 2).contiguous()) * st["scale"]
        if case["cap"]:
            s = case["cap"] * torch.tanh(s / case["cap"])
        nq, nk = qf.shape[1], kf.shape[1]
        at = torch.arange(nk - nq, nk, device=q.device)[:, None]
        j = torch.arange(nk, device=q.device)[None, :]
        if st["slopes"] is not None:
            s = s - st["slopes"][:, None, None] * (at - j).abs().float()
        if case["mask"] != "full":
            s = s.masked_fill((j > at) & (j >= st["prefixes"][b]), float("-inf"))
        p = (s - s.amax(-1, keepdim=True)).exp()
        p = p / p.sum(-1, keepdim=True)
        out.append(torch.matmul(p, vf).transpose(0, 1))
    if tail:
        out.append(torch.zeros((tail, case["heads"], case["width"]), device=q.device))
    return torch.cat(out).to(q.dtype)


def _frequencies(case):
    """(f_i, mag) in 64 bits."""
    R, factor, base = case["turned"], case["factor"], BASE
    i = torch.arange(R // 2, dtype=torch.float64)
    if case["scaling"] == "base":
        base = base * factor ** (R / (R - 2))
    f = base ** (-2.0 * i / R)
    mag = 1.0
    if case["scaling"] == "linear":
        f = f / factor
    elif case["scaling"] == "parts":                          # whole turns within the original length: 32 and more keep f, 1 and less take f / factor
        turns = ORIGINAL * f / (2.0 * math.pi)
        keep = ((turns - 1.0) / 31.0).clamp(0.0, 1.0)
        f = f * keep + f / factor * (1.0 - keep)
        mag = 1.0 + 0.1 * math.log(factor)
    return f, mag


def _plain_rotary(st):
    case, dev = st["case"], st["q"].device
    f, mag = _frequencies(case)
    pos = torch.cat([torch.arange(n, device=dev) + first for n, first in zip(st["lengths"], st["firsts"])])
    angle = pos.double()[:, None] * f.to(dev)
    cos, sin = (angle.cos() * mag).float()[:, None], (angle.sin() * mag).float()[:, None]
    R, n = case["turned"], pos.shape[0]

    def turn(t):
        x = t[:n].float()
        if case["layout"] == "half":
            a, b = x[..., :R // 2], x[..., R // 2:R]
            y = torch.cat([a * cos - b * sin, a * sin + b * cos, x[..., R:]], -1)
        else:
            a, b = x[..., 0:R:2], x[..., 1:R:2]
            y = torch.cat([torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2), x[..., R:]], -1)
        if n < t.shape[0]:
            y = torch.cat([y, torch.zeros_like(t[n:], dtype=torch.float32)])
        return y.to(t.dtype)

    return turn(st["q"]), turn(st["k"])


def _act(z, name):
    if name == "relu":
        return z.clamp_min(0.0)
    if name == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    return z * torch.sigmoid(z) if name == "silu" else z


def _plain_group_norm(st):
    case, x, n = st["case"], st["x"].float(), sum(st["lengths"])
    C, G = case["channels"], case["groups"]
    out = []
    for d in x[:n].split(st["lengths"]):
        d = d.reshape(d.shape[0], G, C // G)
        mean = d.mean((0, 2), keepdim=True)
        centred = d - mean
        var = (centred * centred).mean((0, 2), keepdim=True)
        out.append((centred * torch.rsqrt(var + st["eps"])).reshape(-1, C))
    y = _act(torch.cat(out) * st["w"] + st["b"], case["act"])
    if n < x.shape[0]:
        y = torch.cat([y, torch.zeros_like(x[n:])])
    return y.to(st["x"].dtype)


# ------------------------------------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "attention":
            return _exact_attention(st)
        return _exact_rotary(st) if case["op"] == "rotary" else _exact_group_norm(st)


def _exact_attention(st):
    """Head by head and document by document from the definition, with the gradients written out."""
    case, dev = st["case"], st["q"].device
    group, cap = case["heads"] // case["shared"], case["cap"]
    q, k, v = (st[name].detach().double() for name in ("q", "k", "v"))
    train, token = case["dir"] == "train", case["dir"] == "token"
    o, dq, dk, dv = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    row = 0
    for b, nk in enumerate(st["lengths"]):
        nq = 1 if token else nk
        qr, kr = slice(row, row + nq), slice(b * case["longest"], b * case["longest"] + nk) if token else slice(row, row + nk)
        row += nq
        distance = torch.arange(nk - nq, nk, device=dev)[:, None] - torch.arange(nk, device=dev)[None, :]
        seen = None
        if case["mask"] != "full":
            seen = distance >= 0
            seen[:, :st["prefixes"][b]] = True
        for h in range(case["heads"]):
            qh, kh, vh = q[qr, h], k[kr, h // group], v[kr, h // group]
            x = st["scale"] * (qh @ kh.T)
            if cap:
                t = torch.tanh(x / cap)
                x = cap * t
            if st["slopes"] is not None:
                x = x - st["slopes"][h].double() * distance.abs()
            if seen is not None:
                x = torch.where(seen, x, float("-inf"))
            p = torch.softmax(x, -1)
            o[qr, h] = p @ vh
            if train:
                g = st["do"][qr, h].double()
                dv[kr, h // group] += p.T @ g
                dp = g @ vh.T
                ds = p * (dp - (p * dp).sum(-1, keepdim=True)) * st["scale"]
                if cap:
                    ds = ds * (1.0 - t * t)
                dq[qr, h] = ds @ kh
                dk[kr, h // group] += ds.T @ qh
    return (o, dq, dk, dv) if train else o


def _exact_rotary(st):
    """Each pair as a complex number times mag e^(i angle); the gradient is the product with the conjugate."""
    case, R = st["case"], st["case"]["turned"]
    expo = torch.arange(0, R, 2, dtype=torch.float64, device=st["q"].device) / R
    base, mag = BASE, 1.0
    if case["scaling"] == "base":
        base = BASE * case["factor"] ** (R / (R - 2.0))
    f = torch.exp(-math.log(base) * expo)
    if case["scaling"] == "linear":
        f = f / case["factor"]
    if case["scaling"] == "parts":
        mag = 0.1 * math.log(case["factor"]) + 1.0
        blend = torch.clamp((f * ORIGINAL / (2.0 * math.pi) - 1.0) / (32.0 - 1.0), 0.0, 1.0)
        f = torch.lerp(f / case["factor"], f, blend)
    where = [first + i for n, first in zip(st["lengths"], st["firsts"]) for i in range(n)]
    angle = torch.tensor(where, dtype=torch.float64, device=f.device)[:, None, None] * f
    turn = torch.polar(torch.full_like(angle, mag), angle)
    n = len(where)

    def apply(t, w):
        x = t.detach().double()
        y = torch.zeros_like(x)
        y[:n] = x[:n]
        first, second = (slice(0, R // 2), slice(R // 2, R)) if case["layout"] == "half" else (slice(0, R, 2), slice(1, R, 2))
        z = torch.complex(x[:n, :, first].contiguous(), x[:n, :, second].contiguous()) * w
        y[:n, :, first], y[:n, :, second] = z.real, z.imag
        return y

    out = (apply(st["q"], turn), apply(st["k"], turn))
    return out + (apply(st["dq"], turn.conj()), apply(st["dk"], turn.conj())) if case["dir"] == "train" else out


def _exact_group_norm(st):
    case, x = st["case"], st["x"].detach().double()
    C, G = case["channels"], case["groups"]
    w, b = st["w"].detach().double(), st["b"].detach().double()
    y, dx, dw, db = torch.zeros_like(x), torch.zeros_like(x), torch.zeros_like(w), torch.zeros_like(b)
    row = 0
    for n in st["lengths"]:
        rows = slice(row, row + n)
        row += n
        xg = x[rows].view(n, G, C // G)
        mean = xg.mean((0, 2), keepdim=True)
        rstd = 1.0 / torch.sqrt(((xg - mean) ** 2).mean((0, 2), keepdim=True) + st["eps"])
        hat = ((xg - mean) * rstd).view(n, C)
        z = hat * w + b
        if case["act"] == "silu":
            sg = 1.0 / (1.0 + torch.exp(-z))
            value, slope = z * sg, sg * (1.0 + z * (1.0 - sg))
        elif case["act"] == "gelu":
            cdf = 0.5 * torch.erfc(-z / math.sqrt(2.0))
            value, slope = z * cdf, cdf + z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)
        elif case["act"] == "relu":
            value, slope = torch.where(z > 0, z, torch.zeros_like(z)), (z > 0).double()
        else:
            value, slope = z, torch.ones_like(z)
        y[rows] = value
        if case["dir"] == "train":
            dz = st["dy"][rows].double() * slope
            dw += (dz * hat).sum(0)
            db += dz.sum(0)
            gw = (dz * w).view(n, G, C // G)
            hg = hat.view(n, G, C // G)
            mean_g = gw.mean((0, 2), keepdim=True)
            mean_gh = (gw * hg).mean((0, 2), keepdim=True)
            dx[rows] = (rstd * (gw - mean_g - hg * mean_gh)).view(n, C)
    return (y, dx, dw, db) if case["dir"] == "train" else y
