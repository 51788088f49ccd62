"""Workloads of the language-model operators, as a program calls them.

Four operators: log probabilities of given tokens with entropy and the top
alternatives; distillation from a teacher's top logits with its gradient; linear
attention with a decay for each head, over prompts and single tokens; products
of a few rows with 4-bit weights and group scales.  `run()` computes them in
plain torch, in 32 bits, or, with `own` set, through `pssa_amd`'s entry points
on the same device arrays.  `exact()` has the same results in 64 bits.
"""
from __future__ import annotations

import functools
import math

import torch

own = False

LISTED = [
    # The next token of one stream, over the benchmark's vocabulary, with the alternatives a user sees: latency.
    {"name": "logprobs_1x16384_f32", "op": "logprobs", "rows": 1, "vocab": 16384, "dtype": "f32", "top": 20,
     "temperature": 1.0, "masked": 0.0, "pad": 0},
    # Scoring a batch of 16 chunks of 512 tokens (an evaluation, or a teacher's frames being recorded).
    {"name": "logprobs_8192x16384_f32", "op": "logprobs", "rows": 8192, "vocab": 16384, "dtype": "f32", "top": 8,
     "temperature": 1.0, "masked": 0.0, "pad": 0},
    # A large vocabulary of odd size in bf16, some tokens not allowed, rows in a wider buffer, sampled at 0.7.
    {"name": "logprobs_509x100003_bf16", "op": "logprobs", "rows": 509, "vocab": 100003, "dtype": "bf16", "top": 5,
     "temperature": 0.7, "masked": 0.3, "pad": 29},
    # A student of the reference's small vocabulary on one short chunk: the smallest step.
    {"name": "distill_37x2048_f32", "op": "distill", "rows": 37, "vocab": 2048, "dtype": "f32", "teacher": 8,
     "temperature": 1.0, "pad": 0},
    # A training step of the 105M model: 16 chunks of 512 tokens, 64 teacher logits for each.
    {"name": "distill_8192x16384_f32", "op": "distill", "rows": 8192, "vocab": 16384, "dtype": "f32", "teacher": 64,
     "temperature": 2.0, "pad": 0},
    # A large vocabulary of odd size in bf16, a ragged number of tokens, some of them without weight.
    {"name": "distill_777x65537_bf16", "op": "distill", "rows": 777, "vocab": 65537, "dtype": "bf16", "teacher": 20,
     "temperature": 1.5, "pad": 7},
    # One long prompt, heads of 128 over two shared key heads: few heads, many steps.
    {"name": "linear_1x8192_bf16", "op": "linear", "lens": "8192", "heads": 8, "kv_heads": 2, "d_key": 128, "d_val": 128,
     "dtype": "bf16", "state": False},
    # A batch of prompts at the 105M model's width.
    {"name": "linear_16x1024_bf16", "op": "linear", "lens": ",".join(["1024"] * 16), "heads": 12, "kv_heads": 12,
     "d_key": 64, "d_val": 64, "dtype": "bf16", "state": False},
    # Prompts as they arrive in a server, each continuing its stream's state, in fp32.
    {"name": "linear_ragged_9_f32", "op": "linear", "lens": "817,43,256,611,129,90,377,1000,5", "heads": 12,
     "kv_heads": 12, "d_key": 64, "d_val": 64, "dtype": "f32", "state": True},
    # One token for each of 256 streams: the states pass through once.
    {"name": "linear_step_256_bf16", "op": "linear", "lens": ",".join(["1"] * 256), "heads": 12, "kv_heads": 12,
     "d_key": 64, "d_val": 64, "dtype": "bf16", "state": True},
    # The head of the 105M model for one stream's token.
    {"name": "w4_1x16384x768_bf16", "op": "w4", "rows": 1, "n": 16384, "k": 768, "group": 64, "dtype": "bf16",
     "zeros": False},
    # A wide layer for a few streams, odd row count, fp32 rows, weights with zero points.
    {"name": "w4_7x16384x8192_f32", "op": "w4", "rows": 7, "n": 16384, "k": 8192, "group": 128, "dtype": "f32",
     "zeros": True},
]


def listed():
    return [dict(c) for c in LISTED]


def _log(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["logprobs", "distill", "linear", "linear", "w4"])
    if op in ("logprobs", "distill"):
        vocab = _log(rng, 64, 131072)
        case = {"op": op, "rows": _log(rng, 1, min(8192, 8192 * 16384 // vocab)), "vocab": vocab,
                "dtype": rng.choice(["f32", "bf16"]), "temperature": rng.choice([1.0, 1.0, 0.7, 2.0]),
                "pad": rng.choice([0, 0, 1, 64])}
        if op == "logprobs":
            case.update(top=rng.choice([0, 1, 5, 8, 20, 64]), masked=rng.choice([0.0, 0.0, 0.25]))
        else:
            case.update(teacher=rng.choice([1, 8, 20, 50, 64, 100]))
        case["top" if op == "logprobs" else "teacher"] = min(case.get("top", case.get("teacher")), vocab // 2)
        return case
    if op == "linear":
        kv = rng.choice([1, 2, 4])
        case = {"op": op, "kv_heads": kv, "heads": kv * rng.choice([1, 2, 3]), "d_key": rng.choice([16, 32, 64, 100, 128]),
                "d_val": rng.choice([32, 64, 72, 128, 192]), "dtype": rng.choice(["f32", "bf16", "bf16"]),
                "state": rng.random() < 0.5}
        kind = rng.random()
        if kind < 0.3:  # single tokens
            lens = [1] * _log(rng, 1, 512)
        elif kind < 0.6:  # one prompt
            lens = [_log(rng, 2, 4096)]
        else:  # a ragged batch
            lens = [_log(rng, 1, 1024) for _ in range(rng.randint(2, 12))]
        case["lens"] = ",".join(str(n) for n in lens)
        return case
    return {"op": op, "rows": _log(rng, 1, 32), "n": _log(rng, 64, 16384), "k": _log(rng, 64, 8192),
            "group": rng.choice([32, 64, 128]), "dtype": rng.choice(["f32", "bf16"]), "zeros": rng.random() < 0.5}


# ---------------------------------------------------------------------------
# Inputs.


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _type(case):
    return torch.float32 if case["dtype"] == "f32" else torch.bfloat16


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)


def _randint(g, hi, *shape):
    return torch.randint(0, hi, shape, generator=g, device="cuda")


def _logit_inputs(case, seed):
    """Logits of a trained model: a wide bell with one favoured token a row, from hardly to nearly certain."""
    g, n, v = _gen(seed), case["rows"], case["vocab"]
    wide = _randn(g, n, v + case["pad"]).mul_(2.5)
    best = _randint(g, v, n)
    wide[torch.arange(n, device="cuda"), best] += 18.0 * torch.rand(n, generator=g, device="cuda")
    if case.get("masked"):  # tokens that are not allowed, the favoured one aside
        off = torch.rand(n, v, generator=g, device="cuda") < case["masked"]
        off[torch.arange(n, device="cuda"), best] = False
        wide[:, :v].masked_fill_(off, -math.inf)
    t = {"logits": wide.to(_type(case))}
    if case["op"] == "logprobs":
        # The favoured token, another one, or none (a row behind its sequence's end).
        pick = torch.rand(n, generator=g, device="cuda")
        t["targets"] = torch.where(pick < 0.6, best, torch.where(pick < 0.9, _randint(g, v, n), torch.full_like(best, -1)))
        t["targets"] = t["targets"].to(torch.int32)
        return t
    # A teacher that mostly agrees: distinct tokens, the student's favourite first.
    k = case["teacher"]
    step = _randint(g, max(1, (v - 1) // k), n, 1) + 1
    ids = (best[:, None] + step * torch.arange(k, device="cuda")) % v
    scores = _randn(g, n, k).mul_(2.0)
    scores[:, 0] += 4.0
    dead = torch.rand(n, k, generator=g, device="cuda") < 0.05  # frames with fewer alternatives
    t["ids"] = torch.where(dead, torch.full_like(ids, -1), ids).to(torch.int32)
    t["scores"] = scores
    weights = torch.rand(n, generator=g, device="cuda")
    t["weights"] = torch.where(weights < 0.1, torch.zeros_like(weights), torch.full_like(weights, 1.0 / n))
    return t


def _lens(case):
    return [int(v) for v in case["lens"].split(",")]


def _linear_inputs(case, seed):
    g, lens = _gen(seed), _lens(case)
    h, hk, dk, dv, n = case["heads"], case["kv_heads"], case["d_key"], case["d_val"], sum(lens)
    # One projection's output, as a program has it: a token's queries, keys and values side by side.
    row = _randn(g, n, h * dk + hk * (dk + dv))
    row[:, h * dk:(h + hk) * dk] *= dk ** -0.5
    # Heads remember from some 20 to some 1000 tokens.
    reach = torch.linspace(math.log(20.0), math.log(1000.0), h, dtype=torch.float64, device="cuda").exp()
    state = _randn(g, len(lens), h, dk, dv).mul_(0.5) if case["state"] else None
    return {"row": row.to(_type(case)), "log_decay": torch.log1p(-1.0 / reach).float(), "state": state,
            "scale": dk ** -0.5}


def _w4_inputs(case, seed):
    g, m, n, k = _gen(seed), case["rows"], case["n"], case["k"]
    groups = -(-k // case["group"])
    t = {"x": _randn(g, m, k).to(_type(case)),
         "codes": torch.randint(0, 16, (n, k), generator=g, device="cuda", dtype=torch.uint8),
         "scales": (torch.rand(n, groups, generator=g, device="cuda") + 0.5) * (0.2 / math.sqrt(k)), "zeros": None}
    if case["zeros"]:
        t["zeros"] = torch.randint(5, 12, (n, groups), generator=g, device="cuda", dtype=torch.uint8)
    return t


def _inputs(case, seed):
    if case["op"] in ("logprobs", "distill"):
        return _logit_inputs(case, seed)
    return _linear_inputs(case, seed) if case["op"] == "linear" else _w4_inputs(case, seed)


@functools.lru_cache(maxsize=None)
def _device():
    from pssa_amd import HipDevice

    return HipDevice(0)


def prepare(case, seed):
    st = {"case": dict(case), **_inputs(case, seed)}

    def empty(*shape, dtype=torch.float32):
        return torch.empty(*shape, device="cuda", dtype=dtype)

    if case["op"] == "logprobs":
        n, k = case["rows"], case["top"]
        st["out"] = [empty(n), empty(n)] + ([empty(n, k, dtype=torch.int32), empty(n, k)] if k else [])
    elif case["op"] == "distill":
        st["out"] = [empty(case["rows"]), empty(case["rows"], case["vocab"], dtype=_type(case))]
    elif case["op"] == "linear":
        lens, h, dv = _lens(case), case["heads"], case["d_val"]
        st["out"] = [empty(sum(lens), h, dv, dtype=_type(case)), empty(len(lens), h, case["d_key"], dv)]
        st["lens"] = lens
        st["lens_gpu"] = torch.tensor(lens, device="cuda")
    else:
        st["out"] = empty(case["rows"], case["n"])
    if own:
        st["dev"] = _device()
        if case["op"] == "w4":  # a program keeps the weights in the library's layout
            torch.cuda.synchronize()
            zeros = st["zeros"]
            st["w4"] = st["dev"].w4_matrix_resident(st["codes"].data_ptr(), st["scales"].data_ptr(), case["n"], case["k"],
                                                    case["group"], None if zeros is None else zeros.data_ptr())
        elif case["op"] == "linear":
            st["dev"].linear_attention_reserve(case["dtype"], case["heads"], case["d_key"], case["d_val"], st["lens"])
    torch.cuda.synchronize()
    return st


# ---------------------------------------------------------------------------
# One pass.


def run(state):
    return _run_own(state) if own else _PLAIN[state["case"]["op"]](state)


def _run_own(st):
    case, dev, out = st["case"], st["dev"], st["out"]
    if case["op"] == "logprobs":
        top = case["top"]
        dev.token_logprobs_resident(st["logits"].data_ptr(), case["dtype"], case["rows"], case["vocab"],
                                    st["targets"].data_ptr(), out[0].data_ptr(), out[1].data_ptr(), top,
                                    out[2].data_ptr() if top else None, out[3].data_ptr() if top else None,
                                    temperature=case["temperature"], ld=case["vocab"] + case["pad"])
    elif case["op"] == "distill":
        dev.distill_resident(st["logits"].data_ptr(), case["dtype"], case["rows"], case["vocab"], st["ids"].data_ptr(),
                             st["scores"].data_ptr(), case["teacher"], out[0].data_ptr(), out[1].data_ptr(),
                             temperature=case["temperature"], row_weights_ptr=st["weights"].data_ptr(),
                             ld=case["vocab"] + case["pad"])
    elif case["op"] == "linear":
        row, h, hk, dk, dv = st["row"], case["heads"], case["kv_heads"], case["d_key"], case["d_val"]
        at, size, ld = row.data_ptr(), row.element_size(), row.shape[1]
        dev.linear_attention_resident(at, at + h * dk * size, at + (h + hk) * dk * size, st["log_decay"].data_ptr(),
                                      case["dtype"], h, dk, dv, out[0].data_ptr(), st["lens"], kv_heads=hk,
                                      scale=st["scale"],
                                      state_in_ptr=None if st["state"] is None else st["state"].data_ptr(),
                                      state_out_ptr=out[1].data_ptr(), ld_q=ld, ld_k=ld, ld_v=ld)
    else:
        dev.matvec_w4_resident(st["x"].data_ptr(), case["dtype"], case["rows"], st["w4"], out.data_ptr())
    return out


def _plain_logprobs(st):
    case, v = st["case"], st["case"]["vocab"]
    raw = st["logits"][:, :v].float()
    z = raw / case["temperature"]
    d = z - z.amax(-1, keepdim=True)
    e = torch.exp(d)
    total = e.sum(-1)
    lse = torch.log(total)
    entropy = lse - torch.where(e > 0, e * d, 0.0).sum(-1) / total
    has = st["targets"] >= 0
    given = d.gather(1, st["targets"].clamp_min(0).long()[:, None])[:, 0] - lse
    out = [torch.where(has, given, 0.0), entropy]
    if case["top"]:
        # By logit, then by id: one whole number for both, distinct for every token.
        bits = (raw + 0.0).view(torch.int32)
        order = (bits ^ ((bits >> 31) & 0x7FFFFFFF)).long() * 2 ** 32 + (2 ** 32 - 1 - torch.arange(v, device="cuda"))
        ids = 2 ** 32 - 1 - (order.topk(case["top"], dim=-1).values & (2 ** 32 - 1))
        top = d.gather(1, ids) - lse[:, None]
        out += [torch.where(top > -math.inf, ids, -1).to(torch.int32), top]
    return out


def _plain_distill(st):
    case, v, tau = st["case"], st["case"]["vocab"], st["case"]["temperature"]
    z = st["logits"][:, :v].float() / tau
    d = z - z.amax(-1, keepdim=True)
    e = torch.exp(d)
    total = e.sum(-1, keepdim=True)
    live = st["ids"] >= 0
    ids = st["ids"].clamp_min(0).long()
    t = torch.where(live, st["scores"] / tau, -math.inf)
    t = t - t.amax(-1, keepdim=True)
    et = torch.exp(t)
    q = et / et.sum(-1, keepdim=True)
    log_q = t - torch.log(et.sum(-1, keepdim=True))
    log_p = d.gather(1, ids) - torch.log(total)
    kl = torch.where(q > 0, q * (log_q - log_p), 0.0).sum(-1)
    grad = (e / total).scatter_add_(1, ids, torch.where(live, -q, 0.0))
    w = torch.where(live.any(-1), st["weights"], 0.0)  # a frame without alternatives teaches nothing
    grad = torch.where(w[:, None] > 0, grad, 0.0)
    return [w * tau * tau * kl, (grad * (w * tau)[:, None]).to(_type(case))]


def _split(st):
    """Queries, keys and values [tokens, heads, width] of the token rows, keys and values for every query head."""
    case, row = st["case"], st["row"]
    h, hk, dk, dv, n = case["heads"], case["kv_heads"], case["d_key"], case["d_val"], st["row"].shape[0]
    q = row[:, :h * dk].view(n, h, dk)
    k = row[:, h * dk:(h + hk) * dk].view(n, hk, dk).repeat_interleave(h // hk, 1)
    return q, k, row[:, (h + hk) * dk:].view(n, hk, dv).repeat_interleave(h // hk, 1)


def _plain_linear(st):
    """Every pair of tokens of a sequence: o_t = scale (sum_{j<=t} lambda^(t-j) (q_t k_j) v_j + lambda^(t+1) q_t S)."""
    case, lens = st["case"], st["lens_gpu"]
    n, T = len(st["lens"]), max(st["lens"])
    t = torch.arange(T, device="cuda")
    live = t < lens[:, None]  # [n, T]
    at = ((lens.cumsum(0) - lens)[:, None] + t).clamp_max(st["row"].shape[0] - 1)
    q, k, v = (torch.where(live[:, None, :, None], x.float()[at].transpose(1, 2), 0.0).contiguous() for x in _split(st))
    g = st["log_decay"].double()
    decay = torch.exp((t[:, None] - t).clamp_min(0) * g[:, None, None]).float()
    decay = torch.where(t[:, None] >= t, decay, 0.0)  # [heads, T, T]
    out = torch.matmul(torch.matmul(q, k.transpose(2, 3).contiguous()).mul_(decay), v)
    left = (lens[:, None] - 1 - t).clamp_min(0)  # [n, T]
    kept = torch.exp(left[:, None, :] * g[:, None]).float()[..., None]  # [n, heads, T, 1]
    last = torch.matmul((k * kept).transpose(2, 3).contiguous(), v)
    if st["state"] is not None:
        out = out + torch.matmul(q, st["state"]) * torch.exp((t + 1) * g[:, None]).float()[..., None]
        last = last + st["state"] * torch.exp(lens[:, None] * g).float()[..., None, None]
    return [(out.transpose(1, 2)[live] * st["scale"]).to(_type(case)), last]


def _plain_w4(st):
    case, k, group = st["case"], st["case"]["k"], st["case"]["group"]

    def spread(t):
        return t.float().repeat_interleave(group, 1)[:, :k]

    w = (st["codes"].float() - (8.0 if st["zeros"] is None else spread(st["zeros"]))) * spread(st["scales"])
    return torch.matmul(st["x"].float(), w.T)


_PLAIN = {"logprobs": _plain_logprobs, "distill": _plain_distill, "linear": _plain_linear, "w4": _plain_w4}


# ---------------------------------------------------------------------------
# What a pass cannot do without.


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "logprobs":
        n, v, k = case["rows"], case["vocab"], case["top"]
        return {"bytes": float(n * (v * size + 12 + 8 * k)), "flops": 5.0 * n * v}
    if case["op"] == "distill":
        n, v, k = case["rows"], case["vocab"], case["teacher"]
        return {"bytes": float(n * (2 * v * size + 8 * k + 8)), "flops": 6.0 * n * v}
    if case["op"] == "linear":
        lens, h, hk, dk, dv = _lens(case), case["heads"], case["kv_heads"], case["d_key"], case["d_val"]
        n, state = sum(lens), len(lens) * h * dk * dv * 4
        # The recurrence itself: a state takes 3 operations for its step and 2 for the readout.
        return {"bytes": float(n * (h * (dk + dv) + hk * (dk + dv)) * size + state * (2 if case["state"] else 1) + 4 * h),
                "flops": 5.0 * n * h * dk * dv}
    m, n, k = case["rows"], case["n"], case["k"]
    groups = -(-k // case["group"])
    return {"bytes": n * k / 2.0 + n * groups * (5.0 if case["zeros"] else 4.0) + m * (k * size + n * 4.0),
            "flops": 2.0 * m * n * k}


# ---------------------------------------------------------------------------
# The definitions in 64 bits.


def _exact_logits(case, t, rows):
    """(log softmax, ...) in 64 bits of some rows at the case's temperature."""
    return torch.log_softmax(t["logits"][rows, :case["vocab"]].double() / case["temperature"], -1)


def exact(case, seed):
    t = _inputs(case, seed)
    if case["op"] in ("logprobs", "distill"):
        block = max(1, (1 << 27) // case["vocab"])  # rows at once
        parts = [(_exact_logprobs if case["op"] == "logprobs" else _exact_distill)(case, t, slice(i, i + block))
                 for i in range(0, case["rows"], block)]
        return [None if p[0] is None else torch.cat(p) for p in zip(*parts)]
    return _exact_linear(case, t) if case["op"] == "linear" else _exact_w4(case, t)


def _exact_logprobs(case, t, rows):
    lp = _exact_logits(case, t, rows)
    entropy = torch.special.entr(lp.exp()).sum(-1)
    target = t["targets"][rows].long()
    given = lp[torch.arange(len(target), device="cuda"), target.clamp_min(0)]
    out = [given.masked_fill(target < 0, 0.0), entropy]
    if case["top"]:
        out += [None, lp.sort(-1, descending=True).values[:, :case["top"]].clone()]
    return out


def _exact_distill(case, t, rows):
    tau, lp = case["temperature"], _exact_logits(case, t, rows)
    ids, w = t["ids"][rows].long(), t["weights"][rows].double()
    w[(ids < 0).all(-1)] = 0.0
    ids[:, 0] = torch.where((ids < 0).all(-1), 0, ids[:, 0])
    lq = torch.log_softmax((t["scores"][rows].double() / tau).masked_fill(ids < 0, -math.inf), -1)
    q = lq.exp()
    full = torch.zeros_like(lp).scatter_add(1, ids.clamp_min(0), q)
    cross = -(full * lp).sum(-1)
    return [w * tau ** 2 * (cross - torch.special.entr(q).sum(-1)), (lp.exp() - full) * (w * tau)[:, None]]


def _exact_linear(case, t):
    """The recurrence, token by token: S = lambda S + k v^T, o = scale q S."""
    lens, lam = torch.tensor(_lens(case), device="cuda"), t["log_decay"].double().exp()[:, None, None]
    q, k, v = (x.double() for x in _split({"case": case, "row": t["row"]}))
    n, h, dk, dv = len(lens), case["heads"], case["d_key"], case["d_val"]
    s = torch.zeros(n, h, dk, dv, dtype=torch.float64, device="cuda") if t["state"] is None else t["state"].double()
    out, first = torch.zeros(q.shape[0], h, dv, dtype=torch.float64, device="cuda"), lens.cumsum(0) - lens
    order = torch.argsort(lens, descending=True)  # the longest first: those still running are a prefix
    s, first, sizes = s[order].clone(), first[order], sorted(_lens(case), reverse=True)
    for i in range(sizes[0]):
        while sizes[-1] <= i:
            sizes.pop()
        r = len(sizes)
        at = first[:r] + i
        s[:r].mul_(lam).add_(k[at][..., None] * v[at][..., None, :])
        out[at] = (q[at][..., None] * s[:r]).sum(-2) * t["scale"]
    return [out, s[torch.argsort(order)]]


def _exact_w4(case, t):
    group, k = case["group"], case["k"]
    at = torch.arange(k, device="cuda") // group
    rows, out = 2048, []
    for i in range(0, case["n"], rows):
        sl = slice(i, i + rows)
        zero = 8.0 if t["zeros"] is None else t["zeros"][sl].double()[:, at]
        w = (t["codes"][sl].double() - zero) * t["scales"][sl].double()[:, at]
        out.append(torch.nn.functional.linear(t["x"].double(), w))
    return torch.cat(out, 1)
