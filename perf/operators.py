"""The operators around attention and the experts of a MoE block, in plain form and through the framework.

  attention_bwd    gradients of causal attention from the saved output and log-sum-exp
  rmsnorm_fwd/bwd  RMS norm with the residual's addition, bf16 and / or MXFP8 output
  route_topk/_bwd  routing: scores, balance bias, expert groups, top-k, weights

``own`` false: elementary torch operations in 32 bits (the choice of experts in 64, where scores lie next to one
another), rounded once at the end. ``own`` true: the calls a user makes.
"""
import math

import torch

own = False

HEAD_DIM = 128
EPS = 1e-5


# ---------------------------------------------------------------------------------------------- cases
def _attention(name, batch, seq, q_heads, kv_heads, window=0, softcap=0.0):
    return {"name": name, "op": "attention_bwd", "batch": batch, "seq": seq, "q_heads": q_heads, "kv_heads": kv_heads,
            "window": window, "softcap": softcap}


def _norm(name, rows, hidden, residual, out):
    return {"name": name, "op": "rmsnorm_fwd", "rows": rows, "hidden": hidden, "residual": residual, "out": out}


def _norm_bwd(name, rows, hidden, residual):
    return {"name": name, "op": "rmsnorm_bwd", "rows": rows, "hidden": hidden, "residual": residual}


def _route(name, op, tokens, experts, topk, score, bias=False, groups=1, topk_groups=1, group_score="top2", renormalize=True,
           scale=1.0, dtype="float32", masked=0):
    return {"name": name, "op": op, "tokens": tokens, "experts": experts, "topk": topk, "score": score, "bias": bias,
            "groups": groups, "topk_groups": topk_groups, "group_score": group_score, "renormalize": renormalize,
            "scale": scale, "dtype": dtype, "masked": masked}


def listed():
    return [
        # two short ragged sequences, as in fine-tuning on short answers: launches and latency
        _attention("attention_bwd 2x77", 2, 77, 4, 2),
        # one training sequence of ordinary length at the benchmark's 32 / 8 heads
        _attention("attention_bwd 2048", 1, 2048, 32, 8),
        # a long one: the tensor cores' rate
        _attention("attention_bwd 8192", 1, 8192, 32, 8),
        # sliding window and soft cap, one KV head per query head, a length that no tile divides
        _attention("attention_bwd 2x4001 window cap", 2, 4001, 16, 16, 1000, 30.0),
        # one token of a decode step
        _norm("rmsnorm_fwd 1x2048", 1, 2048, True, "bf16"),
        # a prompt of ordinary length straight into the 8-bit expert path
        _norm("rmsnorm_fwd 1000x5120 mxfp8", 1000, 5120, True, "mxfp8"),
        # the benchmark's token batch in training: bf16 kept for the weight gradients, MXFP8 for the experts
        _norm("rmsnorm_fwd 16384x4096 both", 16384, 4096, True, "both"),
        # gradients at that batch, with the residual stream's own gradient
        _norm_bwd("rmsnorm_bwd 16384x4096", 16384, 4096, True),
        # a small fine-tuning batch of a hidden size that no vector width divides
        _norm_bwd("rmsnorm_bwd 333x1001", 333, 1001, False),
        # the routes of one token
        _route("route_topk 1x64", "route_topk", 1, 64, 8, "softmax"),
        # many experts in groups, chosen with a balance bias
        _route("route_topk 16384x256 groups", "route_topk", 16384, 256, 8, "sigmoid", bias=True, groups=8, topk_groups=4, scale=2.5),
        # the benchmark's 64 experts, 8 a token: gradient of the weights
        _route("route_topk_bwd 16384x64", "route_topk_bwd", 16384, 64, 8, "softmax"),
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(("attention_bwd", "attention_bwd", "rmsnorm_fwd", "rmsnorm_fwd", "rmsnorm_bwd", "route_topk", "route_topk", "route_topk_bwd"))
    if op == "attention_bwd":
        q_heads, kv_heads = rng.choice(((1, 1), (4, 1), (6, 2), (8, 8), (12, 4), (16, 2), (32, 8)))
        # a query that sees one key has no gradient: where every query does, all of dq and dk is rounding
        seq = _log_int(rng, 16, 8192)
        batch = max(1, min(rng.choice((1, 1, 2, 3, 5)), (32 * 8192 * 4096) // (q_heads * seq * max(seq, 1024))))
        case = _attention("", batch, seq, q_heads, kv_heads, rng.choice((0, 0, _log_int(rng, 2, 4096))), rng.choice((0.0, 0.0, 15.0, 50.0)))
    elif op in ("rmsnorm_fwd", "rmsnorm_bwd"):
        rows = _log_int(rng, 1, 32768)
        top = max(128, min(16384, (1 << 26) // rows))
        residual = rng.random() < 0.7
        out = rng.choice(("bf16", "mxfp8", "both")) if op == "rmsnorm_fwd" else "bf16"
        hidden = _log_int(rng, 8, top) if out == "bf16" and rng.random() < 0.5 else 128 * _log_int(rng, 1, top // 128)
        case = _norm("", rows, hidden, residual, out) if op == "rmsnorm_fwd" else _norm_bwd("", rows, hidden, residual)
    else:
        experts, groups = rng.choice(((8, 1), (16, 4), (60, 1), (64, 1), (64, 8), (96, 1), (128, 1), (160, 8), (256, 8), (384, 1), (512, 16)))
        topk_groups = rng.randint(1, groups)
        topk = rng.randint(1, min(16, topk_groups * (experts // groups)))
        score = rng.choice(("softmax", "sigmoid"))
        case = _route("", op, _log_int(rng, 1, (1 << 23) // experts), experts, topk, score, rng.random() < 0.5, groups, topk_groups,
                      rng.choice(("top2", "max")), rng.random() < 0.7, rng.choice((1.0, 2.5)), rng.choice(("float32", "float32", "bfloat16")),
                      rng.choice((0, 0, 1, 3)))
    del case["name"]
    return case


# ---------------------------------------------------------------------------------------------- inputs
def _visible(seq, window, device):
    i = torch.arange(seq, device=device)
    seen = i[:, None] >= i[None, :]
    return seen & (i[:, None] - i[None, :] < window) if window > 0 else seen


def _attention_forward(q, k, v, window, softcap):
    """O (bf16, like q) and the natural-log LSE [batch * q_heads, seq] of the forward pass, a KV head at a time."""
    batch, seq, q_heads, dim = q.shape
    group = q_heads // k.shape[2]
    out = torch.empty_like(q)
    lse = torch.empty((batch, q_heads, seq), dtype=torch.float32, device=q.device)
    hidden = ~_visible(seq, window, q.device)
    for b in range(batch):
        for h in range(k.shape[2]):
            heads = slice(h * group, (h + 1) * group)
            s = q[b, :, heads].float().transpose(0, 1) @ k[b, :, h].float().T / math.sqrt(dim)
            s = softcap * torch.tanh(s / softcap) if softcap > 0 else s
            s.masked_fill_(hidden, -math.inf)
            lse[b, heads] = torch.logsumexp(s, -1)
            out[b, :, heads] = (torch.exp(s - lse[b, heads, :, None]) @ v[b, :, h].float()).transpose(0, 1).to(out.dtype)
    return out, lse.reshape(batch * q_heads, seq)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, dtype=torch.bfloat16):
        return torch.randn(*shape, generator=gen, device="cuda").to(dtype)

    op, state = case["op"], {"case": case}
    if op == "attention_bwd":
        q_shape = (case["batch"], case["seq"], case["q_heads"], HEAD_DIM)
        kv_shape = (case["batch"], case["seq"], case["kv_heads"], HEAD_DIM)
        q, k, v = normal(*q_shape), normal(*kv_shape), normal(*kv_shape)
        out, lse = _attention_forward(q, k, v, case["window"], case["softcap"])
        state.update(q=q, k=k, v=v, out=out, lse=lse, d_out=normal(*q_shape))
    elif op == "rmsnorm_fwd":
        # the residual stream has grown over the layers, the branch's output has not
        state.update(x=normal(case["rows"], case["hidden"]), weight=(1 + 0.1 * normal(case["hidden"], dtype=torch.float32)).bfloat16(),
                     residual=(3 * normal(case["rows"], case["hidden"], dtype=torch.float32)).bfloat16() if case["residual"] else None)
    elif op == "rmsnorm_bwd":
        hidden = (3 * normal(case["rows"], case["hidden"], dtype=torch.float32)).bfloat16()
        state.update(hidden=hidden, rstd=torch.rsqrt(hidden.float().square().mean(-1) + EPS),
                     weight=(1 + 0.1 * normal(case["hidden"], dtype=torch.float32)).bfloat16(), d_y=normal(case["rows"], case["hidden"]),
                     d_hidden=normal(case["rows"], case["hidden"]) if case["residual"] else None)
    else:
        tokens, experts = case["tokens"], case["experts"]
        logits = normal(tokens, experts, dtype=torch.float32)
        if case["masked"]:
            # experts that a token may not use, and now and then a padding token that may use none
            pick = torch.rand(tokens, experts, generator=gen, device="cuda").argsort(-1) < min(case["masked"], experts - 1)
            padding = torch.rand(tokens, 1, generator=gen, device="cuda") < 0.01
            logits = logits.masked_fill(pick | padding, -math.inf)
        state.update(logits=logits.to(getattr(torch, case["dtype"])),
                     bias=0.1 * normal(experts, dtype=torch.float32) if case["bias"] else None)
        if op == "route_topk_bwd":
            state.update(experts=_route_plain(state)["experts"], d_weights=normal(tokens, case["topk"], dtype=torch.float32))
    return state


# ---------------------------------------------------------------------------------------------- plain forms
def _attention_bwd_plain(st):
    c = st["case"]
    batch, seq, q_heads, kv_heads = c["batch"], c["seq"], c["q_heads"], c["kv_heads"]
    group, scale, cap = q_heads // kv_heads, 1.0 / math.sqrt(HEAD_DIM), c["softcap"]
    rows = lambda t: t.float().reshape(batch, seq, kv_heads, -1, HEAD_DIM).permute(0, 2, 3, 1, 4)  # noqa: E731  [B, Hkv, group, S, D]
    q, k, v, do = rows(st["q"]), rows(st["k"]), rows(st["v"]), rows(st["d_out"])
    s = (q @ k.transpose(-1, -2)).mul_(scale)
    if cap > 0:
        t = s.div_(cap).tanh_()
        slope = 1 - t * t
        s = t.mul_(cap)
    p = s.sub_(st["lse"].reshape(batch, kv_heads, group, seq, 1)).exp_().masked_fill_(~_visible(seq, c["window"], q.device), 0.0)
    dv = (p.transpose(-1, -2) @ do).sum(2)
    dp = do @ v.transpose(-1, -2)
    delta = (p * dp).sum(-1, keepdim=True)
    ds = dp.sub_(delta).mul_(p)
    if cap > 0:
        ds = ds.mul_(slope)
    dq = (ds @ k) * scale
    dk = (ds.transpose(-1, -2) @ q).sum(2) * scale
    back = lambda t: t.to(torch.bfloat16)  # noqa: E731
    return {"dq": back(dq.permute(0, 3, 1, 2, 4).reshape(batch, seq, q_heads, HEAD_DIM)), "dk": back(dk.transpose(1, 2)),
            "dv": back(dv.transpose(1, 2))}


def _scale_tensor(e, rows, hidden):
    """Per-block exponents [rows, hidden / 32] -> scale values in the framework's [rows/128, hidden/128, 32, 16] order."""
    e = e.reshape(rows // 128, 4, 32, hidden // 128, 4).permute(0, 3, 2, 1, 4).reshape(rows // 128, hidden // 128, 32, 16)
    return (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def _mxfp8_plain(y):
    """y [T, H] (values of bf16): E4M3 elements [T up to a multiple of 128, H] and their power-of-two scales per 32."""
    rows, hidden = -(-y.shape[0] // 128) * 128, y.shape[1]
    y = torch.cat([y, y.new_zeros(rows - y.shape[0], hidden)]).reshape(rows, hidden // 32, 32)
    mantissa, exponent = torch.frexp(y.abs().amax(-1) / 448)
    e = torch.where(mantissa == 0, -127, (exponent - (mantissa == 0.5).int()).clamp(-127, 127))
    return torch.ldexp(y, -e[..., None]).reshape(rows, hidden).to(torch.float8_e4m3fn), _scale_tensor(e, rows, hidden)


def _rmsnorm_fwd_plain(st):
    c, got = st["case"], {}
    h = st["x"].float()
    if st["residual"] is not None:
        got["hidden"] = (h + st["residual"].float()).to(torch.bfloat16)
        h = got["hidden"].float()
    rstd = torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS)
    y = (h * rstd * st["weight"].float()).to(torch.bfloat16)
    got["rstd"] = rstd[:, 0]
    if c["out"] in ("bf16", "both"):
        got["y"] = y
    if c["out"] in ("mxfp8", "both"):
        got["fp8"], got["scales"] = _mxfp8_plain(y.float())
    return got


def _rmsnorm_bwd_plain(st):
    h, dy, rstd = st["hidden"].float(), st["d_y"].float(), st["rstd"][:, None]
    n = h * rstd
    g = dy * st["weight"].float()
    dx = rstd * (g - n * (g * n).mean(-1, keepdim=True))
    if st["d_hidden"] is not None:
        dx = dx + st["d_hidden"].float()
    return {"dx": dx.to(torch.bfloat16), "d_weight": (dy * n).sum(0)}


def _scores(x, score):
    if score == "sigmoid":
        return 1 / (1 + torch.exp(-x))
    top = x.amax(-1, keepdim=True)
    e = torch.exp(x - torch.where(torch.isinf(top), 0.0, top))
    return e / e.sum(-1, keepdim=True).clamp_min(1e-300)


def _route_plain(st):
    c = st["case"]
    x = st["logits"].double()
    s = _scores(x, c["score"])
    choice = s + st["bias"].double() if st["bias"] is not None else s
    choice = choice.masked_fill(torch.isneginf(x), -math.inf)
    if c["groups"] > 1:
        by_group = choice.reshape(c["tokens"], c["groups"], -1)
        best = by_group.sort(dim=-1, descending=True).values[..., :2 if c["group_score"] == "top2" else 1]
        best = torch.cat([best[..., :1], best[..., 1:].masked_fill(torch.isneginf(best[..., 1:]), 0.0)], -1).sum(-1)
        kept = best.sort(dim=-1, descending=True, stable=True).indices[:, : c["topk_groups"]]
        dropped = torch.ones_like(best, dtype=torch.bool).scatter_(1, kept, False)
        # a masked expert of a kept group still comes before one of a dropped group
        choice = choice.clamp_min(-1e300).reshape(by_group.shape).masked_fill(dropped[..., None], -math.inf).reshape(choice.shape)
    experts = choice.sort(dim=-1, descending=True, stable=True).indices[:, : c["topk"]]
    w = s.gather(1, experts).float()
    if c["renormalize"]:
        total = w.sum(-1, keepdim=True)
        w = torch.where(total > 0, w / total, 0.0)
    return {"experts": experts.int(), "weights": w * c["scale"]}


def _route_bwd_plain(st):
    c = st["case"]
    x, at, g = st["logits"].float(), st["experts"].long(), st["d_weights"] * c["scale"]
    s = _scores(x.double(), c["score"]).float()
    if c["renormalize"]:
        w = s.gather(1, at)
        total = w.sum(-1, keepdim=True)
        g = torch.where(total > 0, (g - (g * w).sum(-1, keepdim=True) / total) / total, 0.0)
    ds = torch.zeros_like(s).scatter_(1, at, g)
    dx = ds * s * (1 - s) if c["score"] == "sigmoid" else s * (ds - (s * ds).sum(-1, keepdim=True))
    return {"d_logits": dx.to(st["logits"].dtype)}


# ---------------------------------------------------------------------------------------------- one pass
def _run_own(st):
    from pipelink_b200 import attention, norm, router
    c = st["case"]
    op = c["op"]
    if op == "attention_bwd":
        dq, dk, dv = attention.attention_bwd(st["d_out"], st["q"], st["k"], st["v"], st["out"], st["lse"], window=c["window"],
                                             softcap=c["softcap"], check=False)
        return {"dq": dq, "dk": dk, "dv": dv}
    if op == "rmsnorm_fwd":
        n = norm.rmsnorm_fwd(st["x"], st["weight"], st["residual"], eps=EPS, out=c["out"])
        got = {"rstd": n.rstd}
        if st["residual"] is not None:
            got["hidden"] = n.hidden
        if n.y is not None:
            got["y"] = n.y
        if n.fp8 is not None:
            got["fp8"], got["scales"] = n.fp8.view(torch.float8_e4m3fn), n.sc.view(torch.float8_e8m0fnu)
        return got
    if op == "rmsnorm_bwd":
        dx, dw = norm.rmsnorm_bwd(st["d_y"], st["hidden"], st["rstd"], st["weight"], st["d_hidden"])
        return {"dx": dx, "d_weight": dw}
    if op == "route_topk":
        experts, weights = router.route_topk(st["logits"], c["topk"], score=c["score"], bias=st["bias"], groups=c["groups"],
                                             topk_groups=c["topk_groups"], group_score=c["group_score"],
                                             renormalize=c["renormalize"], scale=c["scale"])
        return {"experts": experts, "weights": weights}
    return {"d_logits": router.route_topk_bwd(st["d_weights"], st["logits"], st["experts"], score=c["score"],
                                              renormalize=c["renormalize"], scale=c["scale"])}


_PLAIN = {"attention_bwd": _attention_bwd_plain, "rmsnorm_fwd": _rmsnorm_fwd_plain, "rmsnorm_bwd": _rmsnorm_bwd_plain,
          "route_topk": _route_plain, "route_topk_bwd": _route_bwd_plain}


def run(state):
    if own:
        return _run_own(state)
    return _PLAIN[state["case"]["op"]](state)


# ---------------------------------------------------------------------------------------------- 64 bits
def _exact_attention(st):
    """Head by head from the definition: softmax of the visible scores, its Jacobian, the three products."""
    c = st["case"]
    group, scale, cap = c["q_heads"] // c["kv_heads"], HEAD_DIM ** -0.5, c["softcap"]
    dq = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
    dk, dv = (torch.zeros(st["k"].shape, dtype=torch.float64, device="cuda") for _ in range(2))
    seen = _visible(c["seq"], c["window"], "cuda")
    for b in range(c["batch"]):
        for h in range(c["q_heads"]):
            q, k, v, do = st["q"][b, :, h].double(), st["k"][b, :, h // group].double(), st["v"][b, :, h // group].double(), st["d_out"][b, :, h].double()
            x = scale * (q @ k.T)
            y = cap * torch.tanh(x / cap) if cap > 0 else x
            prob = torch.softmax(torch.where(seen, y, -math.inf), dim=-1)
            dv[b, :, h // group] += prob.T @ do
            d_prob = do @ v.T
            d_y = prob * (d_prob - torch.einsum("ij,ij->i", prob, d_prob)[:, None])
            d_x = d_y * (1 - (y / cap) ** 2) if cap > 0 else d_y
            dq[b, :, h] = scale * (d_x @ k)
            dk[b, :, h // group] += scale * (d_x.T @ q)
    return {"dq": dq, "dk": dk, "dv": dv}


def _exact_norm(st):
    c = st["case"]
    h = st["x"].double()
    got = {}
    if st["residual"] is not None:
        h = h + st["residual"].double()
        got["hidden"] = h
        h = h.to(torch.bfloat16).double()          # what is normalised is the stream as it is stored
    got["rstd"] = 1 / torch.sqrt((h * h).sum(-1) / c["hidden"] + EPS)
    y = h * got["rstd"][:, None] * st["weight"].double()
    if c["out"] != "mxfp8":
        got["y"] = y
    if c["out"] != "bf16":
        rows = (c["rows"] + 127) // 128 * 128
        full = torch.zeros(rows, c["hidden"], dtype=torch.float64, device="cuda")
        full[: c["rows"]] = y
        block = full.view(rows, -1, 32)
        largest = block.to(torch.bfloat16).double().abs().amax(-1)
        e = torch.where(largest > 0, torch.ceil(torch.log2(largest.clamp_min(1e-300) / 448)), -127.0).clamp(-127, 127)
        got["fp8"] = (block * torch.exp2(-e)[..., None]).view(rows, -1)
        got["scales"] = torch.exp2(e).view(rows // 128, 4, 32, -1, 4).permute(0, 3, 2, 1, 4).reshape(rows // 128, -1, 32, 16)
    return got


def _exact_norm_bwd(st):
    h, dy, w = st["hidden"].double(), st["d_y"].double(), st["weight"].double()
    size = h.shape[1]
    r = 1 / torch.sqrt((h * h).sum(1) / size + EPS)
    inner = torch.einsum("th,th,h->t", dy, h, w)
    dx = r[:, None] * dy * w - (r ** 3 * inner / size)[:, None] * h
    if st["d_hidden"] is not None:
        dx = dx + st["d_hidden"].double()
    return {"dx": dx, "d_weight": torch.einsum("th,th,t->h", dy, h, r)}


def _exact_scores(st):
    x = st["logits"].double()
    if st["case"]["score"] == "sigmoid":
        return torch.sigmoid(x)
    return torch.nan_to_num(torch.softmax(x, -1), nan=0.0)          # a token that may use no expert


def _exact_route(st):
    c = st["case"]
    s = _exact_scores(st)
    # the choice itself is the plain form's (whole numbers): the weights of those experts
    w = s.gather(1, _route_plain(st)["experts"].long())
    if c["renormalize"]:
        w = torch.nan_to_num(w / w.sum(1, keepdim=True), nan=0.0)
    return {"experts": None, "weights": c["scale"] * w}


def _exact_route_bwd(st):
    c = st["case"]
    at, g = st["experts"].long(), st["d_weights"].double()
    chosen = torch.zeros(c["tokens"], c["topk"], c["experts"], dtype=torch.float64, device="cuda").scatter_(2, at[..., None], 1.0)
    s = _exact_scores(st)
    w = torch.einsum("tke,te->tk", chosen, s)
    if c["renormalize"]:
        total = w.sum(1, keepdim=True)
        jac = torch.diag_embed(1 / total.expand_as(w)) - w[:, None, :] / total[..., None] ** 2     # d w_i / d s_j, transposed
        g = torch.nan_to_num(torch.einsum("tji,ti->tj", jac, g), nan=0.0, posinf=0.0, neginf=0.0)
    d_s = c["scale"] * torch.einsum("tke,tk->te", chosen, g)
    if c["score"] == "sigmoid":
        return {"d_logits": d_s * s * (1 - s)}
    return {"d_logits": s * d_s - s * torch.einsum("te,te->t", s, d_s)[:, None]}


def exact(case, seed):
    st = prepare(case, seed)
    return {"attention_bwd": _exact_attention, "rmsnorm_fwd": _exact_norm, "rmsnorm_bwd": _exact_norm_bwd, "route_topk": _exact_route,
            "route_topk_bwd": _exact_route_bwd}[case["op"]](st)


# ---------------------------------------------------------------------------------------------- work
def work(case):
    op = case["op"]
    if op == "attention_bwd":
        seq, window = case["seq"], case["window"] or case["seq"]
        full = min(seq, window)
        pairs = case["batch"] * case["q_heads"] * (full * (full + 1) // 2 + (seq - full) * full)
        row = case["batch"] * seq * HEAD_DIM * 2
        # q, d_out, out in and dq out; k, v in and dk, dv out; the log-sum-exp; five products over the visible pairs
        return {"bytes": row * 4 * (case["q_heads"] + case["kv_heads"]) + 4 * case["batch"] * seq * case["q_heads"],
                "flops": 5 * 2 * HEAD_DIM * pairs}
    if op == "rmsnorm_fwd":
        n, rows = case["rows"] * case["hidden"], case["rows"]
        got = 2 * n * (1 + 2 * case["residual"]) + 4 * rows + 2 * case["hidden"]
        got += 2 * n * (case["out"] != "mxfp8") + (n + n // 32) * (case["out"] != "bf16")
        return {"bytes": got, "flops": 5 * n}
    if op == "rmsnorm_bwd":
        n = case["rows"] * case["hidden"]
        return {"bytes": 2 * n * (3 + case["residual"]) + 4 * case["rows"] + 6 * case["hidden"], "flops": 10 * n}
    n, size = case["tokens"] * case["experts"], 2 if case["dtype"] == "bfloat16" else 4
    if op == "route_topk":
        return {"bytes": n * size + 8 * case["tokens"] * case["topk"], "flops": 5 * n}
    return {"bytes": 2 * n * size + 8 * case["tokens"] * case["topk"], "flops": 8 * n}
