"""Measured cases of the expert-routing and block-scaled FP8 operators.

Five operators: the router (`moe_gate`), the quantizers that make operands with
a scale per 128 (`quantize_act_fp8`, `quantize_weights_fp8`), the matrix
product of such operands (`matmul_fp8`), the same product grouped by expert
(`matmul_fp8_grouped`) and the expert layer that runs them together
(`moe_fp8`). With `own` false every pass runs the plain form in elementary
torch operations; with `own` true it makes the calls of the mpp41 package.
"""
import math
import os
import sys

import torch

own = False

QMAX = {"e4m3": 448.0, "e5m2": 57344.0}
FP8 = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
OUT = {"f16": torch.float16, "f32": torch.float32}
BLOCK = 128

_ctx = None


def _context():
    """The mpp41 package and one context on torch's stream, as a program keeps them."""
    global _ctx
    if _ctx is None:
        here = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
        sys.path.insert(0, os.path.join(here, "mpp-4.1-fp4-fp8-block_b200"))
        import mpp41
        c = mpp41.Context(torch.cuda.current_device())
        c.set_stream(torch.cuda.current_stream().cuda_stream)
        _ctx = (mpp41, c)
    return _ctx


def _up(n, m):
    return -(-n // m)


# ---------------------------------------------------------------- the cases


def listed():
    return [
        # one decode step of 16 sequences through a 256-expert router: latency
        {"name": "gate_decode", "op": "gate", "tokens": 16, "experts": 256, "top_k": 8, "score": "sigmoid", "bias": True,
         "groups": 8, "top_groups": 4, "group_top": 2, "renormalize": True, "scale": 2.5, "dtype": "f32"},
        # a long prefill through the same router
        {"name": "gate_prefill", "op": "gate", "tokens": 32768, "experts": 256, "top_k": 8, "score": "sigmoid", "bias": True,
         "groups": 8, "top_groups": 4, "group_top": 2, "renormalize": True, "scale": 2.5, "dtype": "f32"},
        # a prefill's activations in front of the experts of the 7168-wide layer
        {"name": "quant_act", "op": "quant_act", "tokens": 4096, "hidden": 7168, "fmt": "e4m3"},
        # a weight matrix of the Llama-3-8B-shaped layer, quantized when it is loaded
        {"name": "quant_weights", "op": "quant_weights", "rows": 14336, "hidden": 4096, "fmt": "e4m3"},
        # one token through that layer's down projection
        {"name": "matmul_decode", "op": "matmul", "m": 1, "n": 4096, "k": 14336, "a": "e4m3", "b": "e4m3", "out": "f16"},
        # a batch of 100 sequences (a ragged tile), fp32 result as for logits or a residual
        {"name": "matmul_batch", "op": "matmul", "m": 100, "n": 14336, "k": 4096, "a": "e4m3", "b": "e4m3", "out": "f32"},
        # prefill through the gate projection
        {"name": "matmul_prefill", "op": "matmul", "m": 4096, "n": 14336, "k": 4096, "a": "e4m3", "b": "e4m3", "out": "f16"},
        # 32 experts of one GPU, 64 tokens' assignments: a few rows an expert, some experts empty
        {"name": "grouped_decode", "op": "grouped", "rows": 512, "used": 500, "groups": 32, "n": 2048, "k": 7168,
         "a": "e4m3", "b": "e4m3", "out": "f16", "skew": 1.0},
        # 2048 tokens' assignments over them
        {"name": "grouped_prefill", "op": "grouped", "rows": 16384, "used": 16384, "groups": 32, "n": 2048, "k": 7168,
         "a": "e4m3", "b": "e4m3", "out": "f16", "skew": 0.5},
        # the expert layer: one token, a decode batch, a prefill chunk
        {"name": "layer_token", "op": "layer", "tokens": 1, "hidden": 7168, "inter": 2048, "experts": 32, "top_k": 8,
         "shared": 2048, "padded": 0, "fmt": "e4m3"},
        {"name": "layer_decode", "op": "layer", "tokens": 128, "hidden": 7168, "inter": 2048, "experts": 32, "top_k": 8,
         "shared": 2048, "padded": 0, "fmt": "e4m3"},
        {"name": "layer_prefill", "op": "layer", "tokens": 2048, "hidden": 7168, "inter": 2048, "experts": 32, "top_k": 8,
         "shared": 0, "padded": 48, "fmt": "e4m3"},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["gate", "quant_act", "quant_weights", "matmul", "matmul", "grouped", "layer"])
    fmt = lambda: rng.choice(["e4m3", "e4m3", "e5m2"])  # noqa: E731
    if op == "gate":
        groups = rng.choice([1, 1, 2, 4, 8, 16])
        experts = groups * rng.randint(2, 512 // groups)
        top_groups = rng.randint(1, groups)
        top_k = rng.randint(1, min(16, experts // groups * top_groups))
        bias = rng.random() < 0.5
        return {"op": op, "tokens": _log(rng, 1, 32768 * 256 // max(256, experts)), "experts": experts, "top_k": top_k,
                "score": rng.choice(["sigmoid", "softmax"]), "bias": bias, "groups": groups, "top_groups": top_groups,
                "group_top": rng.choice([1, 2]), "renormalize": rng.random() < 0.7, "scale": rng.choice([1.0, 2.5]),
                "dtype": rng.choice(["f32", "f32", "f16"])}
    if op == "quant_act":
        hidden = _log(rng, 16, 14336)
        return {"op": op, "tokens": _log(rng, 1, 4096 * 7168 // hidden), "hidden": hidden, "fmt": fmt()}
    if op == "quant_weights":
        hidden = _log(rng, 16, 14336)
        return {"op": op, "rows": _log(rng, 1, min(14336, 14336 * 4096 // hidden)), "hidden": hidden, "fmt": fmt()}
    if op == "matmul":
        n, k = _log(rng, 64, 14336), 16 * _log(rng, 4, 896)
        m = _log(rng, 1, min(8192, 4096 * 14336 * 4096 // (n * k)))
        return {"op": op, "m": m, "n": n, "k": k, "a": fmt(), "b": fmt(), "out": rng.choice(["f16", "f32"])}
    if op == "grouped":
        groups, n, k = rng.randint(1, 48), _log(rng, 64, 2048), 16 * _log(rng, 8, 448)
        rows = _log(rng, 1, 16384)
        used = rows if rng.random() < 0.6 else rng.randint(0, rows)
        return {"op": op, "rows": rows, "used": used, "groups": groups, "n": n, "k": k, "a": fmt(), "b": fmt(),
                "out": rng.choice(["f16", "f32"]), "skew": rng.choice([0.0, 0.5, 1.0, 2.0])}
    hidden, inter = 128 * _log(rng, 4, 56), 128 * _log(rng, 2, 16)
    experts = rng.randint(4, 32)
    tokens = _log(rng, 1, 2048)
    return {"op": op, "tokens": tokens, "hidden": hidden, "inter": inter, "experts": experts,
            "top_k": rng.randint(1, min(8, experts)), "shared": rng.choice([0, 128 * rng.randint(1, 16)]),
            "padded": rng.choice([0, tokens // 8]), "fmt": fmt()}


def work(case):
    c, op = case, case["op"]
    if op == "gate":
        size = 4 if c["dtype"] == "f32" else 2
        return {"bytes": c["tokens"] * (c["experts"] * size + c["top_k"] * 8) + (4 * c["experts"] if c["bias"] else 0),
                "flops": 4.0 * c["tokens"] * c["experts"]}
    if op in ("quant_act", "quant_weights"):
        act = op == "quant_act"
        n = (c["tokens"] if act else c["rows"]) * c["hidden"]
        blocks = (c["tokens"] if act else _up(c["rows"], BLOCK)) * _up(c["hidden"], BLOCK)
        return {"bytes": n * (3 if act else 5) + 4 * blocks, "flops": 2.0 * n}
    if op == "matmul":
        m, n, k = c["m"], c["n"], c["k"]
        return {"bytes": m * k + n * k + m * n * (2 if c["out"] == "f16" else 4) + 4 * _up(k, BLOCK) * (m + _up(n, BLOCK)),
                "flops": 2.0 * m * n * k}
    if op == "grouped":
        m, n, k = c["used"], c["n"], c["k"]
        hit = sum(1 for v in _counts(c) if v)
        return {"bytes": m * k + hit * n * k + m * n * (2 if c["out"] == "f16" else 4) + 4 * _up(k, BLOCK) * (m + hit * _up(n, BLOCK)) +
                4 * (c["groups"] + 1), "flops": max(1.0, 2.0 * m * n * k)}
    rows, h, i = (c["tokens"] - c["padded"]) * c["top_k"], c["hidden"], c["inter"]
    hit = c["experts"] * (1 - (1 - c["top_k"] / c["experts"]) ** (c["tokens"] - c["padded"]))  # experts that some token chooses
    return {"bytes": 3 * h * i * hit + 3 * h * c["shared"] + c["tokens"] * (4 * h + 8 * c["top_k"]),
            "flops": 6.0 * h * (rows * i + c["tokens"] * c["shared"])}


def _counts(c):
    """Rows of each group: shares that fall as a power of the group's place, some groups left empty."""
    g, used = c["groups"], c["used"]
    share = [0.0 if (g > 4 and j % 11 == 5) else (j + 1.0) ** -c["skew"] for j in range(g)]
    share = share[1::2] + share[0::2]
    total = sum(share)
    cum, got = 0.0, []
    for s in share:
        a = int(round(used * cum / total))
        cum += s
        got.append(int(round(used * min(1.0, cum / total))) - a)
    return got


# ---------------------------------------------------------------- inputs


def _blocks_q(w, fmt):
    """fp32 [..., N, K] to 8 bits with a scale per 128 x 128, as a checkpoint has it."""
    lead, (n, k) = w.shape[:-2], w.shape[-2:]
    nb, kb = _up(n, BLOCK), _up(k, BLOCK)
    p = torch.nn.functional.pad(w, (0, kb * BLOCK - k, 0, nb * BLOCK - n)).view(*lead, nb, BLOCK, kb, BLOCK)
    s = (p.abs().amax(dim=(-3, -1)) / QMAX[fmt]).clamp_min(1e-30)
    q = (p / s[..., :, None, :, None]).reshape(*lead, nb * BLOCK, kb * BLOCK)[..., :n, :k]
    return q.clamp(-QMAX[fmt], QMAX[fmt]).to(FP8[fmt]).contiguous(), s.contiguous()


def _rows_q(x, fmt):
    """fp32 [M, K] to 8 bits with a scale per 1 x 128."""
    m, k = x.shape
    kb = _up(k, BLOCK)
    p = torch.nn.functional.pad(x, (0, kb * BLOCK - k)).view(m, kb, BLOCK)
    s = (p.abs().amax(dim=-1) / QMAX[fmt]).clamp_min(1e-30)
    q = (p / s[:, :, None]).reshape(m, kb * BLOCK)[:, :k]
    return q.clamp(-QMAX[fmt], QMAX[fmt]).to(FP8[fmt]).contiguous(), s.contiguous()


def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda")


def _acts(gen, rows, cols):
    """Activations: normal, with some columns far larger, as behind a norm's weight."""
    x = _randn(gen, rows, cols)
    big = torch.rand(cols, generator=gen, device="cuda") < 0.01
    return torch.where(big, x * 20, x)


def prepare(case, seed):
    c, op = case, case["op"]
    gen = torch.Generator(device="cuda").manual_seed(seed * 7919 + 17)
    empty = lambda dt, *shape: torch.empty(*shape, dtype=dt, device="cuda")  # noqa: E731
    st = {"case": dict(c)}
    if op == "gate":
        t, e, k = c["tokens"], c["experts"], c["top_k"]
        st["logits"] = _randn(gen, t, e).to(torch.float32 if c["dtype"] == "f32" else torch.float16)
        st["bias"] = 0.1 * _randn(gen, e) if c["bias"] else None
        st["ids"], st["weights"] = empty(torch.int32, t, k), empty(torch.float32, t, k)
    elif op == "quant_act":
        st["x"] = _acts(gen, c["tokens"], c["hidden"]).half()
        st["q"] = empty(torch.uint8, c["tokens"], c["hidden"])
        st["scales"] = empty(torch.float32, c["tokens"], _up(c["hidden"], BLOCK))
    elif op == "quant_weights":
        st["w"] = 0.02 * _randn(gen, c["rows"], c["hidden"])
        st["q"] = empty(torch.uint8, c["rows"], c["hidden"])
        st["scales"] = empty(torch.float32, _up(c["rows"], BLOCK), _up(c["hidden"], BLOCK))
    elif op == "matmul":
        st["a"], st["sa"] = _rows_q(_acts(gen, c["m"], c["k"]), c["a"])
        st["b"], st["sb"] = _blocks_q(0.02 * _randn(gen, c["n"], c["k"]), c["b"])
        st["c"] = empty(OUT[c["out"]], c["m"], c["n"])
    elif op == "grouped":
        counts = _counts(c)
        cum = [0]
        for v in counts:
            cum.append(cum[-1] + v)
        st["offsets"] = torch.tensor(cum, dtype=torch.int32, device="cuda")
        st["most"] = max(1, max(counts))
        st["a"], st["sa"] = _rows_q(_acts(gen, c["rows"], c["k"]), c["a"])
        st["b"], st["sb"] = _blocks_q(0.02 * _randn(gen, c["groups"], c["n"], c["k"]), c["b"])
        st["c"] = _randn(gen, c["rows"], c["n"]).to(OUT[c["out"]])  # rows behind the last group stay
    else:
        t, h, i, e, s = c["tokens"], c["hidden"], c["inter"], c["experts"], c["shared"]
        st["x"] = _acts(gen, t, h).half()
        logits = _randn(gen, t, e) + 0.5 * _randn(gen, e)  # some experts are asked more than others
        top = torch.sort(logits, dim=1, descending=True, stable=True)
        ids = top.indices[:, :c["top_k"]].to(torch.int32)
        st["weights"] = 2.5 * torch.softmax(top.values[:, :c["top_k"]], dim=1)
        if c["padded"]:  # a padded batch: its last tokens have no expert
            ids[t - c["padded"]:] = -1
        st["ids"] = ids.contiguous()
        st["most"] = max(1, int(torch.bincount(ids[ids >= 0].long(), minlength=1).max())) if t > c["padded"] else 1
        for name, shape in (("wg", (e, i, h)), ("wu", (e, i, h)), ("wd", (e, h, i))):
            st[name], st["s" + name] = _blocks_q(0.02 * _randn(gen, *shape), c["fmt"])
        if s:
            for name, shape in (("hg", (s, h)), ("hu", (s, h)), ("hd", (h, s))):
                st[name], st["s" + name] = _blocks_q(0.02 * _randn(gen, *shape), c["fmt"])
        st["out"] = empty(torch.float16, t, h)
        st["scratch"] = None
    return st


# ---------------------------------------------------------------- the pass


def run(state):
    return (_own if own else _plain)(state)


def _own(st):
    mpp41, ctx = _context()
    c, op = st["case"], st["case"]["op"]
    fmts = {"e4m3": mpp41.FMT_E4M3, "e5m2": mpp41.FMT_E5M2}
    if op == "gate":
        desc = mpp41.gate_desc(c["tokens"], c["experts"], c["top_k"],
                               score=mpp41.GATE_SIGMOID if c["score"] == "sigmoid" else mpp41.GATE_SOFTMAX,
                               groups=c["groups"], top_groups=c["top_groups"], group_top=c["group_top"],
                               renormalize=c["renormalize"], scale=c["scale"], logits_f16=c["dtype"] == "f16")
        ctx.moe_gate(desc, st["logits"], st["bias"], st["ids"], st["weights"])
        return {"ids": st["ids"], "weights": st["weights"]}
    if op == "quant_act":
        ctx.quantize_act_fp8(fmts[c["fmt"]], st["x"], c["tokens"], c["hidden"], st["q"], st["scales"])
        return {"q": st["q"].view(FP8[c["fmt"]]), "scales": st["scales"]}
    if op == "quant_weights":
        ctx.quantize_weights_fp8(fmts[c["fmt"]], st["w"], c["rows"], c["hidden"], st["q"], st["scales"])
        return {"q": st["q"].view(FP8[c["fmt"]]), "scales": st["scales"]}
    if op == "matmul":
        ctx.matmul_fp8(fmts[c["a"]], st["a"], st["sa"], fmts[c["b"]], st["b"], st["sb"], st["c"], c["m"], c["n"], c["k"],
                       c_f16=c["out"] == "f16")
        return st["c"]
    if op == "grouped":
        ctx.matmul_fp8_grouped(fmts[c["a"]], st["a"], st["sa"], fmts[c["b"]], st["b"], st["sb"], st["offsets"], c["groups"],
                               st["c"], c["rows"], c["n"], c["k"], c_f16=c["out"] == "f16")
        return st["c"]
    desc = mpp41.moe_fp8_desc(c["tokens"], c["hidden"], c["inter"], c["experts"], c["top_k"],
                              shared_intermediate=c["shared"], fmt=fmts[c["fmt"]], out_f16=True)
    if st["scratch"] is None:  # kept between passes, as a serving loop keeps it
        st["scratch"] = torch.empty(mpp41.moe_fp8_scratch_bytes(desc), dtype=torch.uint8, device="cuda")
    shared = tuple(st[n] for n in ("hg", "shg", "hu", "shu", "hd", "shd")) if c["shared"] else None
    ctx.moe_fp8(desc, st["x"], st["ids"], st["weights"], st["wg"], st["swg"], st["wu"], st["swu"], st["wd"], st["swd"],
                st["out"], st["scratch"], shared=shared)
    return st["out"]


def _plain_gate(st):
    """Selection in 64 bits, where neighbouring scores are told apart; weights rounded once."""
    c = st["case"]
    t, e, g = c["tokens"], c["experts"], c["groups"]
    z = st["logits"].double()
    s = torch.sigmoid(z) if c["score"] == "sigmoid" else torch.softmax(z, dim=1)
    v = s if st["bias"] is None else s + st["bias"].double()
    if g > 1:
        per = v.view(t, g, e // g)
        n = min(c["group_top"], e // g)
        worth = torch.sort(per, dim=2, descending=True).values[:, :, :n].sum(dim=2)
        keep = torch.sort(worth, dim=1, descending=True, stable=True).indices[:, :c["top_groups"]]
        stays = torch.zeros(t, g, dtype=torch.bool, device=v.device).scatter_(1, keep, True)
        v = per.masked_fill(~stays[:, :, None], -math.inf).reshape(t, e)
    ids = torch.sort(v, dim=1, descending=True, stable=True).indices[:, :c["top_k"]]
    w = torch.gather(s, 1, ids)
    if c["renormalize"]:
        w = w / w.sum(dim=1, keepdim=True)
    return {"ids": ids.to(torch.int32), "weights": (w * c["scale"]).float()}


def _plain_rows(x, fmt):
    """fp32 rows to (8-bit values in fp32, scales [M, kb])."""
    m, k = x.shape
    kb = _up(k, BLOCK)
    p = torch.nn.functional.pad(x, (0, kb * BLOCK - k)).view(m, kb, BLOCK)
    amax = p.abs().amax(dim=2)
    safe = torch.where(amax > 0, amax, torch.ones_like(amax))
    q = (p * QMAX[fmt] / safe[:, :, None]).to(FP8[fmt])
    scale = torch.where(amax > 0, amax / QMAX[fmt], torch.ones_like(amax))
    return q.reshape(m, kb * BLOCK)[:, :k], scale


def _deq_rows(q, s):
    return q.float() * s.repeat_interleave(BLOCK, dim=-1)[..., :q.shape[-1]]


def _deq_blocks(q, s):
    n, k = q.shape[-2:]
    return q.float() * s.repeat_interleave(BLOCK, dim=-2).repeat_interleave(BLOCK, dim=-1)[..., :n, :k]


def _by_group(rows_group, place, a, b, groups, most):
    """Rows of `a` times their group's b[g]^T, each group padded to `most` rows."""
    pad = torch.zeros(groups * most, a.shape[1], device=a.device, dtype=a.dtype)
    pad[rows_group * most + place] = a
    return torch.matmul(pad.view(groups, most, -1), b.transpose(1, 2)).reshape(groups * most, -1)[rows_group * most + place]


def _plain(st):
    c, op = st["case"], st["case"]["op"]
    if op == "gate":
        return _plain_gate(st)
    if op == "quant_act":
        q, s = _plain_rows(st["x"].float(), c["fmt"])
        return {"q": q, "scales": s}
    if op == "quant_weights":
        n, k = c["rows"], c["hidden"]
        nb, kb = _up(n, BLOCK), _up(k, BLOCK)
        p = torch.nn.functional.pad(st["w"], (0, kb * BLOCK - k, 0, nb * BLOCK - n)).view(nb, BLOCK, kb, BLOCK)
        amax = p.abs().amax(dim=(1, 3))
        safe = torch.where(amax > 0, amax, torch.ones_like(amax))
        q = (p / safe[:, None, :, None] * QMAX[c["fmt"]]).to(FP8[c["fmt"]]).reshape(nb * BLOCK, kb * BLOCK)[:n, :k]
        return {"q": q, "scales": torch.where(amax > 0, amax / QMAX[c["fmt"]], torch.ones_like(amax))}
    if op == "matmul":
        return torch.matmul(_deq_rows(st["a"], st["sa"]), _deq_blocks(st["b"], st["sb"]).t()).to(OUT[c["out"]])
    if op == "grouped":
        row = torch.arange(c["rows"], device="cuda")
        group = torch.searchsorted(st["offsets"][1:].long(), row, right=True)
        inside = group < c["groups"]
        group = group.clamp_max(c["groups"] - 1)
        place = torch.where(inside, row - st["offsets"][group], 0)
        a = _deq_rows(st["a"], st["sa"])
        # rows behind the last group go to a place of their own, where nothing reads them
        group = torch.where(inside, group, c["groups"])
        b = torch.cat([_deq_blocks(st["b"], st["sb"]), torch.zeros(1, c["n"], c["k"], device="cuda")])
        y = _by_group(group, place, a, b, c["groups"] + 1, st["most"])
        return torch.where(inside[:, None], y.to(OUT[c["out"]]), st["c"])
    t, k, e = c["tokens"], c["top_k"], c["experts"]
    xq = _deq_rows(*_plain_rows(st["x"].float(), c["fmt"]))
    ids = st["ids"].reshape(-1).long()
    group = torch.where(ids >= 0, ids, e)  # assignments without an expert: a group of zeros
    order = torch.sort(group, stable=True).indices
    counts = torch.zeros(e + 1, dtype=torch.int64, device="cuda").scatter_add_(0, group, torch.ones_like(group))
    start = torch.cumsum(counts, 0) - counts
    place = torch.empty_like(group)
    place[order] = torch.arange(t * k, device="cuda") - start[group[order]]
    place = torch.where(ids >= 0, place, 0)
    zero = lambda w: torch.cat([w, torch.zeros_like(w[:1])])  # noqa: E731
    a = xq.repeat_interleave(k, dim=0)
    gate = _by_group(group, place, a, zero(_deq_blocks(st["wg"], st["swg"])), e + 1, st["most"])
    up = _by_group(group, place, a, zero(_deq_blocks(st["wu"], st["swu"])), e + 1, st["most"])
    mid = _deq_rows(*_plain_rows(gate * torch.sigmoid(gate) * up, c["fmt"]))
    y = _by_group(group, place, mid, zero(_deq_blocks(st["wd"], st["swd"])), e + 1, st["most"])
    y = torch.where((ids >= 0)[:, None], y, torch.zeros_like(y)).view(t, k, -1)
    out = (y * st["weights"][:, :, None]).sum(dim=1)
    if c["shared"]:
        gate, up = (torch.matmul(xq, _deq_blocks(st[n], st["s" + n]).t()) for n in ("hg", "hu"))
        mid = _deq_rows(*_plain_rows(gate * torch.sigmoid(gate) * up, c["fmt"]))
        out = out + torch.matmul(mid, _deq_blocks(st["hd"], st["shd"]).t())
    return out.half()


# ---------------------------------------------------------------- 64 bits


def _wide(q, s, rows_per, cols_per):
    """Values of a block-scaled matrix in 64 bits, each element by its own block's index."""
    n, k = q.shape
    r = torch.arange(n, device=q.device) // rows_per
    d = torch.arange(k, device=q.device) // cols_per
    return q.double() * s.double()[r][:, d]


def _nearest8(x, fmt):
    """Nearest representable 8-bit value (ties to even) of a 64-bit number within range."""
    mant, low = (3, -6) if fmt == "e4m3" else (2, -14)
    _, ex = torch.frexp(x)
    ulp = torch.ldexp(torch.ones_like(x), torch.clamp(ex - 1, min=low) - mant)
    return torch.round(x / ulp) * ulp


def _quant64(x, fmt):
    """A 64-bit matrix, each row in blocks of 128: (8-bit values, scales)."""
    m, k = x.shape
    out, scales = torch.zeros_like(x), []
    for at in range(0, k, BLOCK):
        blk = x[:, at:at + BLOCK]
        amax = blk.abs().max(dim=1).values
        some = amax > 0
        sc = torch.where(some, amax / QMAX[fmt], torch.ones_like(amax))
        out[:, at:at + BLOCK] = torch.where(some[:, None], _nearest8(blk * QMAX[fmt] / torch.where(some, amax, torch.ones_like(amax))[:, None], fmt), 0.0)
        scales.append(sc)
    return out, torch.stack(scales, dim=1)


def exact(case, seed):
    c, op = case, case["op"]
    st = prepare(case, seed)
    if op == "gate":
        t, e, k, g = c["tokens"], c["experts"], c["top_k"], c["groups"]
        z = st["logits"].double()
        if c["score"] == "sigmoid":
            s = 1.0 / (1.0 + torch.exp(-z))
        else:
            x = torch.exp(z - z.max(dim=1, keepdim=True).values)
            s = x / x.sum(dim=1, keepdim=True)
        v = s.clone() if st["bias"] is None else s + st["bias"].double()[None]
        if g > 1:
            size = e // g
            worth = torch.zeros(t, g, dtype=torch.float64, device="cuda")
            for j in range(g):
                blk = v[:, j * size:(j + 1) * size].clone()
                for _ in range(min(c["group_top"], size)):
                    best = blk.max(dim=1)
                    worth[:, j] += best.values
                    blk[torch.arange(t, device="cuda"), best.indices] = -math.inf
            stays = torch.zeros(t, g, dtype=torch.bool, device="cuda")
            for _ in range(c["top_groups"]):
                best = worth == worth.max(dim=1, keepdim=True).values
                first = (best.cumsum(dim=1) == 1) & best
                stays |= first
                worth[first] = -math.inf
            v[~stays.repeat_interleave(size, dim=1)] = -math.inf
        ids = []
        for _ in range(k):
            best = v == v.max(dim=1, keepdim=True).values
            first = ((best.cumsum(dim=1) == 1) & best).double().argmax(dim=1)
            ids.append(first)
            v[torch.arange(t, device="cuda"), first] = -math.inf
        ids = torch.stack(ids, dim=1)
        w = s.gather(1, ids)
        w = w / w.sum(dim=1, keepdim=True) if c["renormalize"] else w
        return {"ids": ids.to(torch.int32), "weights": w * c["scale"]}
    if op == "quant_act":
        q, s = _quant64(st["x"].double(), c["fmt"])
        return {"q": q, "scales": s}
    if op == "quant_weights":
        w = st["w"].double()
        n, k = w.shape
        q, s = torch.zeros_like(w), torch.ones(_up(n, BLOCK), _up(k, BLOCK), dtype=torch.float64, device="cuda")
        for i in range(s.shape[0]):
            strip = w[i * BLOCK:(i + 1) * BLOCK]
            col = torch.nn.functional.pad(strip.abs().max(dim=0).values, (0, s.shape[1] * BLOCK - k)).view(-1, BLOCK).max(dim=1).values
            s[i] = torch.where(col > 0, col / QMAX[c["fmt"]], torch.ones_like(col))
            by = torch.where(col > 0, col, torch.ones_like(col)).repeat_interleave(BLOCK)[:k]
            q[i * BLOCK:(i + 1) * BLOCK] = _nearest8(strip * QMAX[c["fmt"]] / by, c["fmt"])
        return {"q": q, "scales": s}
    if op == "matmul":
        return _wide(st["a"], st["sa"], 1, BLOCK) @ _wide(st["b"], st["sb"], BLOCK, BLOCK).t()
    if op == "grouped":
        y, at = st["c"].double(), 0
        a = _wide(st["a"], st["sa"], 1, BLOCK)
        for g, n in enumerate(_counts(c)):
            if n:
                y[at:at + n] = a[at:at + n] @ _wide(st["b"][g], st["sb"][g], BLOCK, BLOCK).t()
            at += n
        return y
    f = c["fmt"]

    def expert(x, g, sg, u, su, d, sd):
        gate, up = x @ _wide(g, sg, BLOCK, BLOCK).t(), x @ _wide(u, su, BLOCK, BLOCK).t()
        q, s = _quant64(gate / (1.0 + torch.exp(-gate)) * up, f)
        return _wide(q, s, 1, BLOCK) @ _wide(d, sd, BLOCK, BLOCK).t()

    q, s = _quant64(st["x"].double(), f)
    x = _wide(q, s, 1, BLOCK)
    out = expert(x, st["hg"], st["shg"], st["hu"], st["shu"], st["hd"], st["shd"]) if c["shared"] else torch.zeros(c["tokens"], c["hidden"], dtype=torch.float64, device="cuda")
    for e in range(c["experts"]):
        tok, slot = torch.nonzero(st["ids"] == e, as_tuple=True)
        if tok.numel():
            y = expert(x[tok], st["wg"][e], st["swg"][e], st["wu"][e], st["swu"][e], st["wd"][e], st["swd"][e])
            out.index_add_(0, tok, y * st["weights"].double()[tok, slot][:, None])
    return out
