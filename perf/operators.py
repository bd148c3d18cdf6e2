"""What the speed of the packed-batch operators is measured on.

A scene has as many views as it has, a view as many tokens as its image has patches (5 special
tokens and a grid of up to 37 x 37 patches), so batches are packed: the tokens of all scenes one
behind the other, and the bounds of the sequences in ``cu_seqlens``. Kinds of a case:

* ``rotary``: rotary positions with several axes (view, row, column, ...) on q and k together.
* ``rotary_train``: the same and its backward.
* ``attend``: attention within each packed sequence, for inference.
* ``attend_train``: the same and its backward.
* ``paged``: a few new tokens of each sequence over the keys and values kept in a paged cache.

``own`` False computes them from elementary torch operations, True with the framework's operators.
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _rotary(kind, tokens, heads, kv_heads, dim, axes, dtype="bf16", far=64, fused=True):
    """``axes``: dims of each axis, as text; ``far``: positions on the first axis lie below it;
    ``fused``: q and k are column blocks of one projection."""
    return dict(kind=kind, tokens=tokens, heads=heads, kv_heads=kv_heads, dim=dim, axes=axes, dtype=dtype, far=far,
                fused=fused)


def _attend(kind, seqs, shortest, longest, heads, kv_heads, dim, causal, dtype="bf16", spread=0, queries=0):
    """``seqs`` sequences of ``shortest`` to ``longest`` tokens (spread by the number ``spread``);
    ``queries``: query tokens of each sequence, 0 for as many as keys."""
    return dict(kind=kind, seqs=seqs, shortest=shortest, longest=longest, heads=heads, kv_heads=kv_heads, dim=dim,
                causal=causal, dtype=dtype, spread=spread, queries=queries)


def _paged(seqs, shortest, longest, new, heads, kv_heads, dim, page, dtype="bf16", spread=0):
    return dict(kind="paged", seqs=seqs, shortest=shortest, longest=longest, new=new, heads=heads, kv_heads=kv_heads,
                dim=dim, page=page, dtype=dtype, spread=spread)


def listed():
    return [
        # q and k of an image pair's 2 x 1374 tokens, as column blocks of the fused projection.
        dict(_rotary("rotary", 2748, 16, 16, 64, "16,24,24"), name="rotary, 2 views"),
        # A training step's rotation of 48 views with grouped heads of 128.
        dict(_rotary("rotary_train", 48 * 1374, 16, 4, 128, "32,48,48"), name="rotary training, 48 views"),
        # Four axes (scene time, view, row, column), a part of the head left unrotated, odd sizes,
        # frame numbers of a long video, fp32.
        dict(_rotary("rotary_train", 9973, 12, 12, 80, "18,14,20,20", "fp32", 1000000, False), name="rotary training, 4 axes, fp32"),
        # Frame attention: each of four views' tokens among themselves.
        dict(_attend("attend", 4, 1374, 1374, 16, 16, 64, False), name="attention, 4 views"),
        # Global attention over the 32 views of one scene: the largest.
        dict(_attend("attend", 1, 43968, 43968, 16, 16, 64, False), name="attention, 32 views"),
        # Twelve streams of 1 to 9 views in causal order, grouped heads of 128.
        dict(_attend("attend", 12, 1374, 12366, 16, 4, 128, True, "fp16", 1), name="attention, causal streams"),
        # The five special tokens of each of eight scenes over the scene's 2 to 20 views.
        dict(_attend("attend", 8, 2748, 27480, 16, 16, 64, False, "bf16", 2, 5), name="attention, special tokens"),
        # Training on many short ragged sequences (crops), causal.
        dict(_attend("attend_train", 96, 17, 700, 16, 8, 64, True, "bf16", 3), name="attention training, crops"),
        # Training on six scenes of 2 to 8 views.
        dict(_attend("attend_train", 6, 2748, 10992, 16, 16, 64, False, "bf16", 4), name="attention training, scenes"),
        # One new token of one sequence over 4 views: launches and latency.
        dict(_paged(1, 5496, 5496, 1, 16, 16, 64, 64), name="paged, one sequence"),
        # One new token of 64 sequences of 1 to 24 views, grouped heads of 128, small pages.
        dict(_paged(64, 1374, 32976, 1, 32, 8, 128, 16, "bf16", 5), name="paged, 64 sequences"),
        # The five special tokens of a new view of 16 streams over pages that end anywhere.
        dict(_paged(16, 1, 20000, 5, 16, 4, 64, 100, "fp16", 6), name="paged, special tokens"),
    ]


def _log(rng, low, high):
    return min(high, int(low * ((high + 1) / low) ** rng.random()))


def draw(rng):
    kind = rng.choice(["rotary", "rotary_train", "attend", "attend", "attend_train", "attend_train", "paged", "paged"])
    dim = rng.choice([64, 64, 128])
    kv_heads = rng.choice([1, 2, 4, 8, 16])
    heads = kv_heads * rng.choice([g for g in (1, 2, 3, 4, 8) if kv_heads * g <= 32])
    if kind.startswith("rotary"):
        dim = rng.choice([32, 64, 64, 80, 96, 128])
        count = rng.choice([1, 2, 3, 3, 4])
        each = rng.choice([dim // count // 2 * 2, dim // count // 4 * 4, dim // (count + 1) // 2 * 2])
        axes = [each] * (count - 1) + [rng.choice([each, dim - each * (count - 1)])]
        return _rotary(kind, _log(rng, 1, 60000), heads, kv_heads, dim, ",".join(map(str, axes)),
                       rng.choice(["bf16", "bf16", "fp16", "fp32"]), _log(rng, 2, 1000000), rng.random() < 0.5)
    dtype, spread = rng.choice(["bf16", "bf16", "fp16"]), rng.randint(10, 1 << 30)
    if kind == "paged":
        case = _paged(_log(rng, 1, 128), 1, _log(rng, 1, 60000), rng.choice([1, 1, 1, 2, 5, 8]), heads, kv_heads, dim,
                      rng.choice([16, 16, 64, 128, rng.randint(1, 300)]), dtype, spread)
        case["shortest"] = _log(rng, 1, case["longest"])
        limit = 2.0e9
        while work(case)["bytes"] > limit:
            case["seqs"] = (case["seqs"] + 1) // 2
        return case
    train = kind == "attend_train"
    case = _attend(kind, _log(rng, 1, 200), 1, _log(rng, 1, 30000), heads, kv_heads, dim, rng.random() < 0.5, dtype,
                   spread, 0 if train or rng.random() < 0.7 else rng.choice([1, 2, 5, 37, 1374]))
    case["shortest"] = _log(rng, 1, case["longest"])
    # Within the largest listed case, in products and in tokens.
    while work(case)["flops"] > 4.0e12 or sum(_lens(case)) * heads * dim > 48 * 1374 * 2048:
        case["seqs"] = (case["seqs"] + 1) // 2
        if case["seqs"] == 1:
            case["longest"] = max(1, case["longest"] // 2)
            case["shortest"] = min(case["shortest"], case["longest"])
    return case


# ---------------------------------------------------------------------------------------------
# Inputs


def _lens(case):
    """Tokens of each sequence: spread over the logarithm of their range."""
    rng = random.Random(case["spread"])
    return [_log(rng, case["shortest"], case["longest"]) for _ in range(case["seqs"])]


def _query_lens(case):
    return [case["queries"] or n for n in _lens(case)]


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(g, *shape, dtype):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def _bounds(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


def _axes(case):
    return [int(a) for a in case["axes"].split(",")]


def _bases(case):
    return [100.0] * len(_axes(case)) if case["far"] <= 4096 else [10000.0] * len(_axes(case))


def _make(case, seed):
    g, dtype = _gen(seed), DTYPES[case["dtype"]]
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    s = {"case": case}
    if case["kind"].startswith("rotary"):
        t = case["tokens"]
        if case["fused"]:
            y = _randn(g, t, (h + 2 * hk) * d, dtype=dtype)
            s["q"], s["k"] = y[:, :h * d].view(t, h, d), y[:, h * d:(h + hk) * d].view(t, hk, d)
        else:
            s["q"], s["k"] = _randn(g, t, h, d, dtype=dtype), _randn(g, t, hk, d, dtype=dtype)
        tops = [case["far"]] + [38] * (len(_axes(case)) - 1)
        s["pos"] = torch.stack([torch.randint(0, n, (t,), generator=g, device="cuda") for n in tops], -1).to(torch.int32)
        if case["kind"] == "rotary_train":
            s["dq"], s["dk"] = _randn(g, t, h, d, dtype=dtype), _randn(g, t, hk, d, dtype=dtype)
        return s
    if case["kind"] == "paged":
        lens, page = _lens(case), case["page"]
        lens = [max(n, case["new"]) for n in lens]
        pages = [-(-n // page) for n in lens]
        # The pool has some pages to spare, a sequence's pages lie anywhere in it, and the table has
        # room for more pages than any sequence has yet.
        pool, width = sum(pages) + 8, max(pages) + 3
        order = torch.randperm(pool, generator=torch.Generator().manual_seed(int(seed))).to(torch.int32)
        table = torch.full((len(lens), width), -1, dtype=torch.int32)
        at = 0
        for i, n in enumerate(pages):
            table[i, :n] = order[at:at + n]
            at += n
        s["table"], s["lens_host"] = table.cuda(), lens
        s["lens"] = torch.tensor(lens, dtype=torch.int32).cuda()
        s["q"] = _randn(g, len(lens), case["new"], h, d, dtype=dtype) * 1.5
        s["kc"], s["vc"] = (_randn(g, pool, page, hk, d, dtype=dtype) for _ in range(2))
        return s
    lens, qlens = _lens(case), _query_lens(case)
    s["cu_host"], s["cuq_host"] = _bounds(lens), _bounds(qlens)
    s["cu"] = torch.tensor(s["cu_host"], dtype=torch.int32).cuda()
    s["cuq"] = torch.tensor(s["cuq_host"], dtype=torch.int32).cuda()
    s["q"] = _randn(g, sum(qlens), h, d, dtype=dtype) * 1.5
    s["k"], s["v"] = (_randn(g, sum(lens), hk, d, dtype=dtype) for _ in range(2))
    if case["kind"] == "attend_train":
        s["do"] = _randn(g, sum(qlens), h, d, dtype=dtype)
    return s


def prepare(case, seed):
    s = _make(case, seed)
    names = {"rotary_train": ("q", "k"), "attend_train": ("q", "k", "v")}.get(case["kind"], ())
    for n in names:
        s[n] = s[n].detach().requires_grad_(own)
    return s


# ---------------------------------------------------------------------------------------------
# One pass


def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    case = s["case"]
    kind = case["kind"]
    if kind.startswith("rotary"):
        from geoweave_amd.rotary import rotary_axes_qk_func

        q, k = rotary_axes_qk_func(s["q"], s["k"], s["pos"], _axes(case), _bases(case))
        if kind == "rotary":
            return {"q": q, "k": k}
        dq, dk = torch.autograd.grad([q, k], [s["q"], s["k"]], [s["dq"], s["dk"]])
        return {"q": q.detach(), "k": k.detach(), "dq": dq, "dk": dk}
    if kind == "paged":
        from geoweave_amd.custom_flash_attn.paged_flash_attn import paged_flash_attn_inference_func

        o, _ = paged_flash_attn_inference_func(s["q"], s["kc"], s["vc"], s["table"], s["lens"])
        return {"o": o}
    from geoweave_amd.custom_flash_attn.packed_flash_attn import (packed_flash_attn_func,
                                                                  packed_flash_attn_inference_func)

    if kind == "attend":
        o, _ = packed_flash_attn_inference_func(s["q"], s["k"], s["v"], s["cuq"], s["cu"], causal=case["causal"])
        return {"o": o}
    o = packed_flash_attn_func(s["q"], s["k"], s["v"], s["cuq"], s["cu"], case["causal"])
    dq, dk, dv = torch.autograd.grad(o, [s["q"], s["k"], s["v"]], s["do"])
    return {"o": o.detach(), "dq": dq, "dk": dk, "dv": dv}


def _rotate(x, pos, axes, bases, sign):
    """x [T, H, D] in fp32; the angles in 64 bits."""
    parts, at = [], 0
    for a, (n, base) in enumerate(zip(axes, bases)):
        freq = base ** (-torch.arange(0, n, 2, device=x.device, dtype=torch.float64) / n)
        t = pos[:, a].double()[:, None] * freq
        cos, sin = t.cos().float()[:, None], (sign * t.sin()).float()[:, None]
        x1, x2 = x[..., at:at + n // 2], x[..., at + n // 2:at + n]
        parts += [x1 * cos - x2 * sin, x2 * cos + x1 * sin]
        at += n
    return torch.cat(parts + [x[..., at:]], dim=-1)


def _rows(heads, keys):
    """Query rows at a time, so that a block's scores stay within about 1 GiB of fp32."""
    return max(1, (1 << 28) // (heads * max(keys, 1)))


def _allowed(a, b, lq, lk, causal, device):
    if not causal:
        return None
    i = torch.arange(a, b, device=device)[:, None] + (lk - lq)
    return torch.arange(lk, device=device)[None] <= i


def _weights(q, k, scale, allowed):
    """q [H, n, D], k [H, L, D] -> softmax weights [H, n, L]; a row that sees no key has none."""
    t = torch.matmul(q, k.transpose(1, 2)) * scale
    if allowed is not None:
        t = t.masked_fill(~allowed, -math.inf)
    top = t.amax(-1, keepdim=True)
    t = (t - torch.where(top == -math.inf, torch.zeros_like(top), top)).exp()
    total = t.sum(-1, keepdim=True)
    return t / torch.where(total == 0, torch.ones_like(total), total)


def _heads(x, times):
    """[L, H, D] -> fp32 [H * times, L, D], each head ``times`` times."""
    return x.float().transpose(0, 1).repeat_interleave(times, 0)


def _plain_attend(q, k, v, causal):
    """One sequence: q [Lq, Hq, D], k, v [Lk, Hk, D] -> fp32 [Lq, Hq, D]."""
    lq, h, d = q.shape
    lk, hk = k.shape[:2]
    if lk == 0:
        return torch.zeros(lq, h, d, device=q.device)
    qh, kh, vh = _heads(q, 1), _heads(k, h // hk), _heads(v, h // hk)
    step, out = _rows(h, lk), []
    for a in range(0, lq, step):
        b = min(a + step, lq)
        w = _weights(qh[:, a:b], kh, d ** -0.5, _allowed(a, b, lq, lk, causal, q.device))
        out.append(torch.matmul(w, vh).transpose(0, 1))
    return torch.cat(out)


def _plain_attend_backward(q, k, v, do, causal):
    lq, h, d = q.shape
    lk, hk = k.shape[:2]
    g, scale = h // hk, d ** -0.5
    qh, kh, vh, doh = _heads(q, 1), _heads(k, g), _heads(v, g), _heads(do, 1)
    dk, dv = torch.zeros_like(kh), torch.zeros_like(vh)
    step, dq, out = _rows(h, lk) // 2 + 1, [], []
    for a in range(0, lq, step):
        b = min(a + step, lq)
        w = _weights(qh[:, a:b], kh, scale, _allowed(a, b, lq, lk, causal, q.device))
        o = torch.matmul(w, vh)
        dw = torch.matmul(doh[:, a:b], vh.transpose(1, 2))
        ds = w * (dw - (o * doh[:, a:b]).sum(-1, keepdim=True)) * scale
        dq.append(torch.matmul(ds, kh).transpose(0, 1))
        dk += torch.matmul(ds.transpose(1, 2), qh[:, a:b])
        dv += torch.matmul(w.transpose(1, 2), doh[:, a:b])
        out.append(o.transpose(0, 1))
    fold = lambda t: t.view(hk, g, lk, d).sum(1).transpose(0, 1)  # noqa: E731
    return torch.cat(out), torch.cat(dq), fold(dk), fold(dv)


def _run_plain(s):
    case = s["case"]
    kind, dtype = case["kind"], DTYPES[case["dtype"]]
    if kind.startswith("rotary"):
        axes, bases = _axes(case), _bases(case)
        out = {n: _rotate(s[n].float(), s["pos"], axes, bases, 1.0).to(dtype) for n in ("q", "k")}
        if kind == "rotary_train":
            out.update({n: _rotate(s[n].float(), s["pos"], axes, bases, -1.0).to(dtype) for n in ("dq", "dk")})
        return out
    if kind == "paged":
        out = []
        for i, n in enumerate(s["lens_host"]):
            rows = s["table"][i, :-(-n // case["page"])].long()
            k, v = (s[c][rows].flatten(0, 1)[:n] for c in ("kc", "vc"))
            out.append(_plain_attend(s["q"][i], k, v, True))
        return {"o": torch.stack(out).to(dtype)}
    outs = []
    for i in range(case["seqs"]):
        a, b, c, e = *s["cuq_host"][i:i + 2], *s["cu_host"][i:i + 2]
        q, k, v = s["q"][a:b], s["k"][c:e], s["v"][c:e]
        if kind == "attend":
            outs.append((_plain_attend(q, k, v, case["causal"]),))
        else:
            outs.append(_plain_attend_backward(q, k, v, s["do"][a:b], case["causal"]))
    return dict(zip(("o", "dq", "dk", "dv"), (torch.cat(t).to(dtype) for t in zip(*outs))))


# ---------------------------------------------------------------------------------------------
# What a pass cannot do without


def work(case):
    """Inputs read once, outputs written once, and the products over the pairs that count."""
    size = 4 if case["dtype"] == "fp32" else 2
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    if case["kind"].startswith("rotary"):
        passes = 2 if case["kind"] == "rotary_train" else 1
        t, turned = case["tokens"], sum(_axes(case))
        return {"bytes": passes * (2 * t * (h + hk) * d * size + 4 * t * len(_axes(case))),
                "flops": passes * 3 * t * (h + hk) * turned}
    lens = _lens(case)
    if case["kind"] == "paged":
        new = case["new"]
        lens = [max(n, new) for n in lens]
        pairs = sum(new * n - new * (new - 1) // 2 for n in lens)
        pages = sum(-(-n // case["page"]) for n in lens)
        return {"bytes": 2 * sum(lens) * hk * d * size + 2 * len(lens) * new * h * d * size + 4 * (pages + len(lens)),
                "flops": 4 * d * h * pairs}
    pairs = 0
    for lq, lk in zip(_query_lens(case), lens):
        if not case["causal"]:
            pairs += lq * lk
        else:  # query i sees the first i + lk - lq + 1 keys
            n = min(lq, lk)
            pairs += n * lk - n * (n - 1) // 2
    tq, tk = sum(_query_lens(case)), sum(lens)
    q_bytes, k_bytes = tq * h * d * size, tk * hk * d * size
    if case["kind"] == "attend":
        return {"bytes": 2 * q_bytes + 2 * k_bytes, "flops": 4 * d * h * pairs}
    # the forward's two products and the backward's five; q, do, o, dq and k, v, dk, dv
    return {"bytes": 4 * q_bytes + 4 * k_bytes, "flops": 14 * d * h * pairs}


# ---------------------------------------------------------------------------------------------
# The same in 64 bits, from the definitions


def _exact_head(q, k, v, do, causal, scale):
    """One head of one sequence in 64 bits: q, do [Lq, D], k, v [Lk, D]."""
    lq, lk = q.shape[0], k.shape[0]
    o, dq, dk, dv = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    step = max(1, (1 << 27) // max(lk, 1))
    for a in range(0, lq, step):
        c = slice(a, min(a + step, lq))
        t = (q[c] @ k.t()) * scale
        if causal:
            row = torch.arange(c.start, c.stop, device=q.device)[:, None]
            t[torch.arange(lk, device=q.device)[None] > row + lk - lq] = -math.inf
        p = torch.exp(t - torch.logsumexp(t, 1, keepdim=True).clamp_min(-1e300))
        del t
        o[c] = p @ v
        if do is not None:
            dp = do[c] @ v.t()
            ds = p * (dp - (p * dp).sum(1, keepdim=True))
            dq[c] = scale * (ds @ k)
            dk += scale * (ds.t() @ q[c])
            dv += p.t() @ do[c]
    return o, dq, dk, dv


def _exact_sequence(q, k, v, do, causal):
    h, hk, scale = q.shape[1], k.shape[1], 1.0 / math.sqrt(q.shape[2])
    o, dq = torch.zeros_like(q, dtype=torch.float64), torch.zeros_like(q, dtype=torch.float64)
    dk, dv = torch.zeros_like(k, dtype=torch.float64), torch.zeros_like(v, dtype=torch.float64)
    for i in range(h):
        j = i * hk // h
        r = _exact_head(q[:, i].double(), k[:, j].double(), v[:, j].double(),
                        None if do is None else do[:, i].double(), causal, scale)
        o[:, i], dq[:, i] = r[0], r[1]
        dk[:, j] += r[2]
        dv[:, j] += r[3]
    return o, dq, dk, dv


def _exact_rotary(x, pos, axes, bases, sign):
    """Pair (x1, x2) as the complex number x1 + i x2, turned by exp(i angle)."""
    x = x.double()
    y, at = x.clone(), 0
    for a, n in enumerate(axes):
        half = n // 2
        i = torch.arange(half, device=x.device, dtype=torch.float64)
        angle = sign * pos[:, a].double()[:, None] / torch.pow(torch.tensor(bases[a], device=x.device, dtype=torch.float64), 2 * i / n)
        z = torch.complex(x[..., at:at + half], x[..., at + half:at + n]) * torch.polar(torch.ones_like(angle), angle)[:, None]
        y[..., at:at + half], y[..., at + half:at + n] = z.real, z.imag
        at += n
    return y


def exact(case, seed):
    s = _make(case, seed)
    kind = case["kind"]
    if kind.startswith("rotary"):
        names = (("q", 1.0), ("k", 1.0)) + ((("dq", -1.0), ("dk", -1.0)) if kind == "rotary_train" else ())
        return {n: _exact_rotary(s[n], s["pos"], _axes(case), _bases(case), sign) for n, sign in names}
    if kind == "paged":
        out = []
        for i, n in enumerate(s["lens_host"]):
            at = torch.arange(n, device="cuda")
            page = s["table"][i].long()[at // case["page"]]
            k, v = (s[c][page, at % case["page"]] for c in ("kc", "vc"))
            out.append(_exact_sequence(s["q"][i], k, v, None, True)[0])
        return {"o": torch.stack(out)}
    outs = []
    for i in range(case["seqs"]):
        a, b, c, e = *s["cuq_host"][i:i + 2], *s["cu_host"][i:i + 2]
        outs.append(_exact_sequence(s["q"][a:b], s["k"][c:e], s["v"][c:e], s["do"][a:b] if "do" in s else None, case["causal"]))
    names = ("o", "dq", "dk", "dv") if kind == "attend_train" else ("o",)
    return dict(zip(names, (torch.cat(t) for t in zip(*outs))))
