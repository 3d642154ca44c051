"""The operators around a language model's output distribution, as cases to be measured.

Two operators over logits [rows, V] (row stride `ld`, fp32 or bf16), with z = scale * logits, scale the inverse
temperature, and p = softmax(z):

  token log probabilities   logp[r] = z[r, token] - lse(z[r]), the entropy of p[r], and the `top` most likely
                            classes with their log probabilities; backward: the gradients of logp and of the entropy
  top-k distillation        loss[r] = KL(q || p) where q is given by a teacher's `top` logits (softmax over them) or
                            log probabilities (all other classes are then one more class, "tail"), with its gradient

`own` chooses what run() does: the plain form in elementary torch operations, or the calls of this package's C ABI.
"""
import functools
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
NO_TOKEN = -1            # a position without a token, an alternative or a teacher slot that does not exist


def listed():
    def case(name, op, dtype, rows, vocab, ld=0, top=0, entropy=True, masked=0.0, scale=1.0, tail=False):
        return {"name": name, "op": op, "dtype": dtype, "rows": rows, "vocab": vocab, "ld": ld or vocab, "top": top,
                "entropy": entropy, "masked": masked, "scale": scale, "tail": tail}

    return [
        # one generated token of one request, with the alternatives an answer shows
        case("logprobs: one token", "logprobs", "bf16", 1, 128256, top=20, entropy=False),
        # a decode batch whose grammar leaves a tenth of the classes
        case("logprobs: masked batch", "logprobs", "bf16", 48, 151936, top=8, masked=0.9),
        # an odd batch over a vocabulary padded to a multiple of 64, at temperature 0.7
        case("logprobs: padded vocabulary", "logprobs", "f32", 37, 50257, ld=50304, top=5, scale=1 / 0.7),
        # scoring sequences: perplexity, ranking, the old policy's log probabilities
        case("logprobs: scoring", "logprobs", "f32", 4096, 50257),
        # a teacher writes its top logits down for a batch of sequences
        case("logprobs: teacher top 64", "logprobs", "bf16", 8192, 128256, top=64, entropy=False),
        # a policy gradient with an entropy bonus, odd row length
        case("logprobs backward: odd rows", "logprobs_backward", "bf16", 2048, 50257, scale=1 / 0.9),
        # the same for a batch of long sequences
        case("logprobs backward: batch", "logprobs_backward", "f32", 4096, 128256),
        # the loss of a held-out batch, without a gradient
        case("distill: evaluation", "distill", "f32", 512, 32768, top=16),
        # a student's training step: loss and gradient of a batch, teacher logits softened
        case("distill step: 32 of 32768", "distill_step", "f32", 8192, 32768, top=32, scale=0.5),
        # the same with the teacher's remaining mass as one more class
        case("distill step: 64 of 151936, tail", "distill_step", "bf16", 8192, 151936, top=64, tail=True),
        # long fp32 rows
        case("distill step: 100 of 128256, tail", "distill_step", "f32", 2048, 128256, top=100, tail=True),
        # loss and gradient as two nodes of a graph: the upstream gradient comes from what follows the loss
        case("distill graph: odd rows", "distill_graph", "bf16", 2048, 50257, top=20, tail=True),
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["logprobs", "logprobs", "logprobs_backward", "distill", "distill_step", "distill_graph"])
    dtype = rng.choice(["f32", "bf16"])
    vocab = spread(257, 151936)
    vocab = vocab if rng.random() < 0.5 else max(256, vocab // 64 * 64)
    ld = vocab if rng.random() < 0.7 else (vocab // 64 + 1) * 64
    most = int(1.2e9 // vocab) if dtype == "bf16" else int(0.5e9 // vocab)
    rows = spread(1, max(2, min(32768, most)))
    lists = op.startswith("distill")
    top = spread(1, 128) if lists or rng.random() < 0.7 else 0
    return {"op": op, "dtype": dtype, "rows": rows, "vocab": vocab, "ld": ld, "top": 0 if op == "logprobs_backward" else top,
            "entropy": rng.random() < 0.5, "masked": rng.choice([0.0, 0.0, 0.5, 0.95]) if op == "logprobs" else 0.0,
            "scale": rng.choice([1.0, 1.0, 0.5, 1.25]), "tail": lists and rng.random() < 0.5}


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _student(c, g):
    """logits with a few likely classes in each row, the rest a broad bulk"""
    rows, V, ld = c["rows"], c["vocab"], c["ld"]
    x = torch.randn(rows, ld, device="cuda", generator=g).mul_(2.2)
    x += torch.randn(rows, 1, device="cuda", generator=g)
    likely = torch.randint(0, V, (rows, 12), device="cuda", generator=g)
    x.scatter_add_(1, likely, 6.0 + 3.0 * torch.rand(rows, 12, device="cuda", generator=g))
    if c["masked"]:
        x[torch.rand(rows, ld, device="cuda", generator=g) < c["masked"]] = -math.inf
        x[:, min(7, V - 1)] = 1.0                   # (a grammar leaves at least one class)
    return x, likely


def _teacher(c, g):
    """distinct ids a row, values descending; some rows have fewer slots, a few are padding without any"""
    rows, V, K = c["rows"], c["vocab"], c["top"]
    K_ids = min(K, V)
    start = torch.randint(0, V, (rows, 1), device="cuda", generator=g)
    step = torch.randint(1, V // K_ids + 1, (rows, 1), device="cuda", generator=g)
    k = torch.arange(K, device="cuda")[None]
    ids = (start + k * step) % V
    values = torch.sort(3.0 * torch.randn(rows, K, device="cuda", generator=g), dim=1, descending=True).values
    if c["tail"]:
        rest = values.amax(1, keepdim=True) - 1.0 - 2.0 * torch.rand(rows, 1, device="cuda", generator=g)
        both = torch.cat([values, rest], 1).double()
        values = (both - both.exp().sum(1, keepdim=True).log())[:, :K].float()
    u = torch.rand(rows, 1, device="cuda", generator=g)
    u[0] = 1.0
    used = torch.where(u < 0.05, 0, torch.where(u < 0.15, (K + 1) // 2, K))
    ids = torch.where(k < torch.clamp(used, max=V), ids, NO_TOKEN)
    return ids.to(torch.int32).contiguous(), values.contiguous()


def prepare(case, seed):
    c, g = case, _generator(seed)
    rows, V, K = c["rows"], c["vocab"], c["top"]
    dtype = DTYPES[c["dtype"]]
    x, likely = _student(c, g)
    s = {"case": c}

    def empty(*shape, dtype=torch.float32):
        return torch.zeros(*shape, dtype=dtype, device="cuda")

    if c["op"].startswith("logprobs"):
        sampled = likely[:, 0]
        anywhere = torch.randint(0, V, (rows,), device="cuda", generator=g)
        u = torch.rand(rows, device="cuda", generator=g)
        tokens = torch.where(u < 0.7, sampled, anywhere)
        s["tokens"] = torch.where((u > 0.97) & (torch.arange(rows, device="cuda") > 0), NO_TOKEN, tokens).to(torch.int32)
    else:
        s["teacher_ids"], s["teacher_values"] = _teacher(c, g)
        # the student knows something of what its teacher says
        x.scatter_add_(1, s["teacher_ids"].clamp(min=0).long(), 0.7 * s["teacher_values"].clamp(min=-6) * (s["teacher_ids"] >= 0))
    s["logits"] = x.to(dtype)
    del x
    if c["op"] == "logprobs":
        s["logp"], s["lse"] = empty(rows), empty(rows)
        s["entropy"] = empty(rows) if c["entropy"] else None
        s["top_ids"] = empty(rows, K, dtype=torch.int32) if K else None
        s["top_logp"] = empty(rows, K) if K else None
    elif c["op"] == "logprobs_backward":
        # what the forward pass left
        lse, ent = [], []
        for part in s["logits"][:, :V].split(1024):
            z = part.double() * _rounded(c["scale"])
            top = z.amax(1, keepdim=True)
            e = (z - top).exp()
            total = e.sum(1, keepdim=True)
            lse.append((top + total.log())[:, 0].float())
            ent.append((total.log() - (e * (z - top)).sum(1, keepdim=True) / total)[:, 0].float())
        s["lse"], s["entropy"] = torch.cat(lse), torch.cat(ent)
        s["dlogp"] = torch.randn(rows, device="cuda", generator=g) / rows
        s["dentropy"] = 0.01 * torch.rand(rows, device="cuda", generator=g) / rows if c["entropy"] else None
        s["dlogits"] = torch.zeros_like(s["logits"])
    else:
        s["loss"] = empty(rows)
        s["stats"] = empty(rows, 4)
        s["weight"] = torch.rand(rows, device="cuda", generator=g) / rows
        if c["op"] != "distill":
            s["dlogits"] = torch.zeros_like(s["logits"])
    return s


def _rounded(scale):
    """the scale that a call with a float argument takes"""
    return torch.tensor(scale, dtype=torch.float32).item()


# ---- plain forms ---------------------------------------------------------------------------------
def _soft(z):
    """(shift, exp(z - shift), their sum) of each row"""
    m = z.amax(1, keepdim=True)
    shift = torch.where(torch.isinf(m), 0.0, m)
    e = torch.exp(z - shift)
    return shift, e, e.sum(1, keepdim=True)


def _plain_logprobs(s):
    c = s["case"]
    V, K, tokens = c["vocab"], c["top"], s["tokens"].long()
    z = s["logits"][:, :V].float() * _rounded(c["scale"])
    shift, e, total = _soft(z)
    log_total = total.log()
    at = z.gather(1, tokens.clamp(min=0)[:, None])
    out = {"logp": torch.where(tokens >= 0, ((at - shift) - log_total)[:, 0], 0.0), "lse": (shift + log_total)[:, 0]}
    if c["entropy"]:
        out["entropy"] = (log_total - (e * torch.where(e > 0, z - shift, 0.0)).sum(1, keepdim=True) / total)[:, 0]
    if K:
        # one whole number a class that orders by the logit, then by the lower index
        raw = (s["logits"][:, :V].float() + 0.0).view(torch.int32)          # (-0 ties with 0)
        order = (raw ^ ((raw >> 31) & 0x7FFFFFFF)).long()
        key = (order << 32) + (V - 1 - torch.arange(V, device=raw.device))
        found = V - 1 - (torch.topk(key, min(K, V), dim=1).values & 0xFFFFFFFF)
        value = z.gather(1, found)
        there = value > -math.inf
        pad = (0, K - found.shape[1])
        out["top_ids"] = torch.nn.functional.pad(torch.where(there, found, NO_TOKEN), pad, value=NO_TOKEN).to(torch.int32)
        out["top_logp"] = torch.nn.functional.pad(torch.where(there, (value - shift) - log_total, -math.inf), pad, value=-math.inf)
    return out


def _plain_logprobs_backward(s):
    c = s["case"]
    V, tokens, scale = c["vocab"], s["tokens"].long(), _rounded(c["scale"])
    logp = s["logits"][:, :V].float() * scale - s["lse"][:, None]
    p = logp.exp()
    g = torch.where(tokens >= 0, s["dlogp"], 0.0)[:, None]
    d = -g * p
    if s["dentropy"] is not None:
        d = d - s["dentropy"][:, None] * p * (torch.where(p > 0, logp, 0.0) + s["entropy"][:, None])
    d.scatter_add_(1, tokens.clamp(min=0)[:, None], g)
    return {"dlogits": (d * scale).to(s["logits"].dtype)}


def _plain_distill(s, gradient):
    c = s["case"]
    V, scale = c["vocab"], _rounded(c["scale"])
    ids, there = s["teacher_ids"].clamp(min=0).long(), s["teacher_ids"] >= 0
    w = torch.where(there, s["teacher_values"] * (1.0 if c["tail"] else scale), -math.inf)
    any_slot = there.any(1, keepdim=True)
    if c["tail"]:
        log_q = w
    else:
        top, e, total = _soft(w)
        log_q = torch.where(any_slot, (w - top) - total.log(), -math.inf)
    q = log_q.exp()
    z = s["logits"][:, :V].float() * scale
    shift, e, total = _soft(z)
    log_total = total.log()
    at = (z.gather(1, ids) - shift) - log_total
    loss = torch.where(q > 0, q * (log_q - at), 0.0).sum(1, keepdim=True)
    in_set = torch.zeros_like(z, dtype=torch.int32).scatter_add_(1, ids, there.int()) > 0
    if c["tail"]:
        q_rest = (1.0 - q.sum(1, keepdim=True)).clamp(min=0.0)
        p_rest = torch.where(in_set, 0.0, e).sum(1, keepdim=True) / total
        has_rest = (q_rest > 0) & (p_rest > 0)
        loss = loss + torch.where(has_rest, q_rest * (q_rest.log() - p_rest.log()), 0.0)
        mass = q.sum(1, keepdim=True) + torch.where(has_rest, q_rest, 0.0)
        outside = mass - torch.where(has_rest, q_rest / p_rest, 0.0)
    else:
        mass = any_slot.float()
        outside = mass
    out = {"loss": loss[:, 0]}
    if gradient:
        d = (e / total) * torch.where(in_set, mass, outside)
        d.scatter_add_(1, ids, torch.where(there, -q, 0.0))
        out["dlogits"] = (d * (s["weight"][:, None] * scale)).to(s["logits"].dtype)
    return out


# ---- the framework's calls -----------------------------------------------------------------------
@functools.lru_cache(maxsize=None)
def _context():
    from autograd_amd import capi
    return capi.Context(0), capi


def _ptr(t):
    return None if t is None else t.data_ptr()


def _own_logprobs(s):
    c = s["case"]
    ctx, capi = _context()
    kind = capi.F32 if c["dtype"] == "f32" else capi.BF16
    ctx.call("agrad_token_logprobs_forward", kind, _ptr(s["logits"]), _ptr(s["tokens"]), _ptr(s["logp"]), _ptr(s["entropy"]),
             _ptr(s["lse"]), _ptr(s["top_ids"]), _ptr(s["top_logp"]), c["rows"], c["vocab"], c["ld"], c["top"], c["scale"])
    return {k: s[k] for k in ("logp", "lse", "entropy", "top_ids", "top_logp") if s[k] is not None}


def _own_logprobs_backward(s):
    c = s["case"]
    ctx, capi = _context()
    kind = capi.F32 if c["dtype"] == "f32" else capi.BF16
    ctx.call("agrad_token_logprobs_backward", kind, _ptr(s["logits"]), _ptr(s["tokens"]), _ptr(s["lse"]), _ptr(s["entropy"]),
             _ptr(s["dlogp"]), _ptr(s["dentropy"]), _ptr(s["dlogits"]), c["rows"], c["vocab"], c["ld"], c["scale"], 0)
    return {"dlogits": s["dlogits"][:, :c["vocab"]]}


def _own_distill(s):
    c = s["case"]
    ctx, capi = _context()
    kind = capi.F32 if c["dtype"] == "f32" else capi.BF16
    mode = capi.DISTILL_TAIL if c["tail"] else capi.DISTILL_RENORM
    soft = 1.0 if c["tail"] else c["scale"]
    shape = (c["rows"], c["vocab"], c["ld"], c["top"], c["scale"], soft)
    if c["op"] == "distill_step":
        ctx.call("agrad_topk_distill_fused", kind, _ptr(s["logits"]), _ptr(s["teacher_ids"]), _ptr(s["teacher_values"]),
                 _ptr(s["loss"]), _ptr(s["weight"]), _ptr(s["dlogits"]), *shape, 1.0, mode)
    else:
        ctx.call("agrad_topk_distill_forward", kind, _ptr(s["logits"]), _ptr(s["teacher_ids"]), _ptr(s["teacher_values"]),
                 _ptr(s["loss"]), _ptr(s["stats"]), *shape, mode)
    if c["op"] == "distill_graph":
        ctx.call("agrad_topk_distill_backward", kind, _ptr(s["logits"]), _ptr(s["teacher_ids"]), _ptr(s["teacher_values"]),
                 _ptr(s["weight"]), _ptr(s["stats"]), _ptr(s["dlogits"]), *shape, mode, 0)
    if c["op"] == "distill":
        return {"loss": s["loss"]}
    return {"loss": s["loss"], "dlogits": s["dlogits"][:, :c["vocab"]]}


def run(state):
    op = state["case"]["op"]
    if own:
        return {"logprobs": _own_logprobs, "logprobs_backward": _own_logprobs_backward}.get(op, _own_distill)(state)
    if op == "logprobs":
        return _plain_logprobs(state)
    if op == "logprobs_backward":
        return _plain_logprobs_backward(state)
    return _plain_distill(state, op != "distill")


def work(case):
    c = case
    e = 4 if c["dtype"] == "f32" else 2
    n = c["rows"] * c["vocab"]
    if c["op"] == "logprobs":
        outs = 2 + int(c["entropy"]) + 2 * c["top"]
        return {"bytes": n * e + 4 * c["rows"] * (1 + outs), "flops": n * (4 + 2 * int(c["entropy"]))}
    if c["op"] == "logprobs_backward":
        return {"bytes": 2 * n * e + 4 * c["rows"] * (3 + 2 * int(c["entropy"])), "flops": n * (4 + 2 * int(c["entropy"]))}
    lists = 8 * c["rows"] * c["top"]
    if c["op"] == "distill":
        return {"bytes": n * e + lists + 4 * c["rows"], "flops": 4 * n}
    return {"bytes": 2 * n * e + lists + 8 * c["rows"], "flops": 6 * n}


# ---- 64 bits -------------------------------------------------------------------------------------
def exact(case, seed):
    """the definitions, a block of rows at a time"""
    s, c = prepare(case, seed), case
    V, K, scale, tail = c["vocab"], c["top"], _rounded(c["scale"]), c["tail"]
    parts = {}

    def keep(name, value):
        parts.setdefault(name, []).append(value)

    block = max(1, (1 << 27) // V)
    for lo in range(0, c["rows"], block):
        rows = slice(lo, min(lo + block, c["rows"]))
        z = s["logits"][rows, :V].double() * scale
        lse = torch.logsumexp(z, 1)
        logp = z - lse[:, None]
        p = logp.exp()
        plogp = torch.where(p > 0, p * logp, 0.0)
        if c["op"].startswith("logprobs"):
            t = s["tokens"][rows].long()
            asked = t >= 0
            here = torch.arange(V, device=z.device)[None] == t[:, None]
            if c["op"] == "logprobs":
                keep("logp", torch.where(asked, logp.gather(1, t.clamp(min=0)[:, None])[:, 0], 0.0))
                keep("lse", lse)
                if c["entropy"]:
                    keep("entropy", -plogp.sum(1))
                if K:
                    # (which classes come first is whole numbers: only their values are computed here)
                    v = torch.topk(logp, min(K, V), dim=1).values
                    keep("top_logp", torch.cat([v, v.new_full((v.shape[0], K - v.shape[1]), -math.inf)], 1))
            else:
                d = s["dlogp"][rows].double()[:, None] * asked[:, None] * (here.double() - p)
                if s["dentropy"] is not None:
                    h = -plogp.sum(1, keepdim=True)
                    d = d - s["dentropy"][rows].double()[:, None] * (plogp + p * h)
                keep("dlogits", d * scale)
            continue
        ids, used = s["teacher_ids"][rows].long(), s["teacher_ids"][rows] >= 0
        values = s["teacher_values"][rows].double()
        if tail:
            q = torch.where(used, values.exp(), 0.0)
        else:
            q = torch.where(used, torch.softmax(torch.where(used, values * scale, -1e300), 1), 0.0)
        onto = torch.zeros_like(z).scatter_add_(1, ids.clamp(min=0), q)
        member = torch.zeros_like(z).scatter_add_(1, ids.clamp(min=0), used.double()) > 0
        loss = torch.where(q > 0, q * (q.log() - logp.gather(1, ids.clamp(min=0))), 0.0).sum(1)
        d = p * q.sum(1, keepdim=True) - onto
        if tail:
            q_rest = (1.0 - q.sum(1)).clamp(min=0.0)
            p_rest = torch.where(member, 0.0, p).sum(1)
            some = (q_rest > 0) & (p_rest > 0)
            loss = loss + torch.where(some, q_rest * (q_rest.log() - p_rest.log()), 0.0)
            ratio = torch.where(some, q_rest / p_rest, 0.0)
            d = d + torch.where(some, q_rest, 0.0)[:, None] * p - torch.where(member, 0.0, ratio[:, None] * p)
        keep("loss", loss)
        if c["op"] != "distill":
            keep("dlogits", d * (s["weight"][rows].double() * scale)[:, None])
    out = {k: torch.cat(v) for k, v in parts.items()}
    if c["op"] == "logprobs" and K:
        out["top_ids"] = None
    return out
