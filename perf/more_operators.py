"""Workloads of a recurrent language model's serving step, as a program calls them.

Four operators: the root-mean-square norm with the residual's addition, its rows
as they are or in 8 bits with a scale for each; products of 8-bit rows and
weights with scales for each row and channel; the gated delta rule over prompts
and single tokens; the selection of beam search, which reorders the states.
`run()` computes them in plain torch, in 32 bits (64 where neighbouring scores
are told apart and where a triangular matrix is inverted), or, with `own` set,
through `pssa_amd`'s entry points on the same device arrays.  `exact()` has the
same results in 64 bits.
"""
from __future__ import annotations

import functools
import math

import torch

own = False

EOS = 2  # the token that ends a beam

LISTED = [
    # One token for each of 256 streams at the 105M model's width: latency.
    {"name": "norm_256x768_f32", "op": "norm", "rows": 256, "width": 768, "dtype": "f32", "residual": True, "pad": 0},
    # The residual stream of 8192 prompt tokens of a wide model.
    {"name": "norm_8192x8192_bf16", "op": "norm", "rows": 8192, "width": 8192, "dtype": "bf16", "residual": True, "pad": 0},
    # A prompt's tokens through the norm and the projection behind it, all in 8 bits; odd counts, rows in wider buffers.
    {"name": "norm_i8_1021x4100_n5003_bf16", "op": "norm_i8", "rows": 1021, "width": 4100, "n": 5003, "dtype": "bf16",
     "residual": True, "pad": 12, "out": "bf16"},
    # The head of the 105M model for one stream's token.
    {"name": "i8_1x16384x768_f32", "op": "i8", "m": 1, "n": 16384, "k": 768, "out": "f32", "pad": 0},
    # A wide layer for the tokens of 24 streams: the weights pass once.
    {"name": "i8_24x8192x8192_f32", "op": "i8", "m": 24, "n": 8192, "k": 8192, "out": "f32", "pad": 0},
    # The same layer over 8192 prompt tokens.
    {"name": "i8_8192x8192x8192_bf16", "op": "i8", "m": 8192, "n": 8192, "k": 8192, "out": "bf16", "pad": 0},
    # One long prompt, 8 heads of 128 over 4 heads of queries and keys: few heads, many steps.
    {"name": "delta_1x8192_bf16", "op": "delta", "lens": "8192", "heads": 8, "key_heads": 4, "d_key": 128, "d_val": 128,
     "dtype": "bf16", "state": False},
    # A batch of prompts at the 105M model's width.
    {"name": "delta_16x1024_bf16", "op": "delta", "lens": ",".join(["1024"] * 16), "heads": 12, "key_heads": 12,
     "d_key": 64, "d_val": 64, "dtype": "bf16", "state": False},
    # Prompts as they arrive in a server, each continuing its stream's state, in fp32.
    {"name": "delta_ragged_9_f32", "op": "delta", "lens": "817,43,256,611,129,90,377,1000,5", "heads": 12,
     "key_heads": 12, "d_key": 64, "d_val": 64, "dtype": "f32", "state": True},
    # One token for each of 256 streams: the states pass through once.
    {"name": "delta_step_256_bf16", "op": "delta", "lens": ",".join(["1"] * 256), "heads": 12, "key_heads": 12,
     "d_key": 64, "d_val": 64, "dtype": "bf16", "state": True},
    # One request with 4 beams over the benchmark's vocabulary, states of 12 heads of 64 x 64: latency.
    {"name": "beam_1x4x16384_f32", "op": "beam", "groups": 1, "beams": 4, "vocab": 16384, "keep": 4, "dtype": "f32",
     "masked": 0.0, "pad": 0, "words": 49152},
    # 64 requests with 8 beams over a large vocabulary of odd size in bf16, some tokens not allowed, some beams ended.
    {"name": "beam_64x8x100003_bf16", "op": "beam", "groups": 64, "beams": 8, "vocab": 100003, "keep": 8,
     "dtype": "bf16", "masked": 0.3, "pad": 29, "words": 49152},
]


def listed():
    return [dict(c) for c in LISTED]


def _log(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["norm", "norm_i8", "i8", "delta", "delta", "beam"])
    if op == "norm":
        width = _log(rng, 16, 16384)
        return {"op": op, "rows": _log(rng, 1, min(16384, 8192 * 8192 // width)), "width": width,
                "dtype": rng.choice(["f32", "bf16", "bf16"]), "residual": rng.random() < 0.7, "pad": rng.choice([0, 0, 1, 64])}
    if op == "norm_i8":
        return {"op": op, "rows": _log(rng, 1, 4096), "width": _log(rng, 64, 8192), "n": _log(rng, 64, 8192),
                "dtype": rng.choice(["f32", "bf16"]), "residual": rng.random() < 0.5, "pad": rng.choice([0, 0, 12]),
                "out": rng.choice(["f32", "bf16"])}
    if op == "i8":
        n, k = _log(rng, 32, 16384), _log(rng, 32, 16384)
        return {"op": op, "m": _log(rng, 1, min(8192, 8192 ** 3 // (n * k))), "n": n, "k": k,
                "out": rng.choice(["f32", "bf16"]), "pad": rng.choice([0, 0, 1, 16])}
    if op == "delta":
        keys = rng.choice([1, 2, 4])
        case = {"op": op, "key_heads": keys, "heads": keys * rng.choice([1, 2, 3]), "d_key": rng.choice([16, 32, 64, 100, 128]),
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
    vocab, beams = _log(rng, 128, 131072), rng.choice([1, 2, 4, 5, 8, 16])
    return {"op": op, "groups": _log(rng, 1, max(1, min(128, 512 * 100003 // (vocab * beams)))), "beams": beams,
            "vocab": vocab, "keep": rng.choice([beams, beams, 2 * beams]), "dtype": rng.choice(["f32", "bf16"]),
            "masked": rng.choice([0.0, 0.0, 0.25]), "pad": rng.choice([0, 0, 1, 64]), "words": _log(rng, 16, 16384)}


# ---------------------------------------------------------------------------
# Inputs.


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _type(name):
    return torch.float32 if name == "f32" else torch.bfloat16


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)


def _rand(g, *shape):
    return torch.rand(*shape, generator=g, device="cuda", dtype=torch.float32)


def _i8(g, n, k):
    """Codes of a normal distribution whose largest value is about 127, as a row's or a channel's scale leaves them."""
    return _randn(g, n, k).mul_(32.0).round_().clamp_(-127, 127).to(torch.int8)


def _norm_inputs(case, seed):
    g, n, d, p = _gen(seed), case["rows"], case["width"], case["pad"]
    # A residual stream: some channels are far wider than the others, and rows of different size.
    wide = 1.0 + 7.0 * (_rand(g, d + p) < 0.02)
    t = {"x": (_randn(g, n, d + p) * wide * (0.5 + _rand(g, n, 1))).to(_type(case["dtype"])),
         "gamma": 1.0 + 0.2 * _randn(g, d), "residual": None}
    if case["residual"]:
        t["residual"] = _randn(g, n, d + p).to(_type(case["dtype"]))
    if case["op"] == "norm_i8":
        t["w"] = _i8(g, case["n"], d)
        t["w_scales"] = (0.5 + _rand(g, case["n"])) * (3.0 / 127.0) / math.sqrt(d)
    return t


def _i8_inputs(case, seed):
    g, m, n, k, p = _gen(seed), case["m"], case["n"], case["k"], case["pad"]
    return {"x": _i8(g, m, k + p), "x_scales": (0.5 + _rand(g, m)) * (4.0 / 127.0), "w": _i8(g, n, k + p),
            "w_scales": (0.5 + _rand(g, n)) * (3.0 / 127.0) / math.sqrt(k)}


def _lens(case):
    return [int(v) for v in case["lens"].split(",")]


def _delta_inputs(case, seed):
    g, lens = _gen(seed), _lens(case)
    h, hk, dk, dv, n = case["heads"], case["key_heads"], case["d_key"], case["d_val"], sum(lens)
    # Queries and keys of length one; a head's keys share a direction (a cosine of about 0.2 between any two).
    q, k = _randn(g, n, hk, dk), _randn(g, n, hk, dk) + 0.5 * _randn(g, 1, hk, dk)
    q, k = (t / t.norm(dim=-1, keepdim=True) for t in (q, k))
    row = torch.cat([q.reshape(n, -1), k.reshape(n, -1), _randn(g, n, h * dv)], 1)
    # A token's gates side by side: decays from hardly any to e^-1 or so, and half-way updates.
    pace = torch.linspace(math.log(0.003), math.log(0.5), h, device="cuda").exp()
    decay = -pace * torch.log1p(torch.exp(_randn(g, n, h)))
    gates = torch.cat([decay, torch.sigmoid(_randn(g, n, h))], 1)
    state = _randn(g, len(lens), h, dk, dv).mul_(0.5) if case["state"] else None
    return {"row": row.to(_type(case["dtype"])), "gates": gates, "state": state, "scale": dk ** -0.5}


def _beam_inputs(case, seed):
    g, n, v = _gen(seed), case["groups"] * case["beams"], case["vocab"]
    logits = _randn(g, n, v + case["pad"]).mul_(2.5)
    if case["masked"]:  # tokens that are not allowed
        logits[:, :v].masked_fill_(_rand(g, n, v) < case["masked"], -math.inf)
    last = torch.randint(EOS + 1, v, (case["groups"], case["beams"]), generator=g, device="cuda")
    ended = _rand(g, case["groups"], case["beams"]) < 0.1
    ended[:, 0] = False
    return {"logits": logits.to(_type(case["dtype"])), "last": torch.where(ended, EOS, last).to(torch.int32),
            "scores": -20.0 + 2.0 * _randn(g, case["groups"], case["beams"]), "states": _randn(g, n, case["words"])}


_INPUTS = {"norm": _norm_inputs, "norm_i8": _norm_inputs, "i8": _i8_inputs, "delta": _delta_inputs, "beam": _beam_inputs}


@functools.lru_cache(maxsize=None)
def _device():
    from pssa_amd import HipDevice

    return HipDevice(0)


def prepare(case, seed):
    st = {"case": dict(case), **_INPUTS[case["op"]](case, seed)}

    def empty(*shape, dtype=torch.float32):
        return torch.empty(*shape, device="cuda", dtype=dtype)

    if case["op"] in ("norm", "norm_i8"):
        n, d, t = case["rows"], case["width"], _type(case["dtype"])
        st["out"] = [empty(n, d, dtype=t)] if case["residual"] else []
        if case["op"] == "norm":
            st["out"].append(empty(n, d, dtype=t))
        else:
            st["codes"], st["scales"] = empty(n, d, dtype=torch.int8), empty(n)
            st["out"].append(empty(n, case["n"], dtype=_type(case["out"])))
    elif case["op"] == "i8":
        st["out"] = empty(case["m"], case["n"], dtype=_type(case["out"]))
    elif case["op"] == "delta":
        lens, h, dv = _lens(case), case["heads"], case["d_val"]
        st["out"] = [empty(sum(lens), h, dv, dtype=_type(case["dtype"])), empty(len(lens), h, case["d_key"], dv)]
        st["lens"], st["lens_gpu"] = lens, torch.tensor(lens, device="cuda")
    else:
        g, k = case["groups"], case["keep"]
        st["out"] = [empty(g, k, dtype=torch.int32), empty(g, k, dtype=torch.int32), empty(g, k), empty(g * k, case["words"])]
    if own:
        st["dev"] = _device()
        if case["op"] == "i8":
            st["dev"].matmul_i8_reserve(case["m"], case["n"], case["k"])
        elif case["op"] == "norm_i8":
            st["dev"].matmul_i8_reserve(case["rows"], case["n"], case["width"])
        elif case["op"] == "delta":
            st["dev"].delta_rule_reserve(case["dtype"], case["heads"], case["d_key"], case["d_val"], st["lens"])
        elif case["op"] == "beam":
            st["dev"].beam_select_reserve(case["groups"], case["beams"], case["vocab"], case["keep"])
    torch.cuda.synchronize()
    return st


# ---------------------------------------------------------------------------
# One pass.


def run(state):
    return _run_own(state) if own else _PLAIN[state["case"]["op"]](state)


def _run_own(st):
    case, dev, out = st["case"], st["dev"], st["out"]
    if case["op"] in ("norm", "norm_i8"):
        d, ld, q = case["width"], case["width"] + case["pad"], case["op"] == "norm_i8"
        res = st["residual"]
        dev.rms_norm_resident(st["x"].data_ptr(), case["dtype"], case["rows"], d, st["gamma"].data_ptr(),
                              residual_ptr=None if res is None else res.data_ptr(),
                              sum_ptr=None if res is None else out[0].data_ptr(),
                              out_ptr=None if q else out[-1].data_ptr(), codes_ptr=st["codes"].data_ptr() if q else None,
                              scales_ptr=st["scales"].data_ptr() if q else None, eps=1e-5, ld_x=ld, ld_residual=ld)
        if q:
            dev.matmul_i8_resident(st["codes"].data_ptr(), st["scales"].data_ptr(), st["w"].data_ptr(),
                                   st["w_scales"].data_ptr(), case["rows"], case["n"], d, out[-1].data_ptr(), case["out"])
    elif case["op"] == "i8":
        ld = case["k"] + case["pad"]
        dev.matmul_i8_resident(st["x"].data_ptr(), st["x_scales"].data_ptr(), st["w"].data_ptr(),
                               st["w_scales"].data_ptr(), case["m"], case["n"], case["k"], out.data_ptr(), case["out"],
                               ld_x=ld, ld_w=ld)
    elif case["op"] == "delta":
        row, h, hk, dk, dv = st["row"], case["heads"], case["key_heads"], case["d_key"], case["d_val"]
        at, size, ld, gates = row.data_ptr(), row.element_size(), row.shape[1], st["gates"].data_ptr()
        dev.delta_rule_resident(at, at + hk * dk * size, at + 2 * hk * dk * size, gates, gates + 4 * h, case["dtype"], h,
                                dk, dv, out[0].data_ptr(), st["lens"], key_heads=hk, scale=st["scale"],
                                state_in_ptr=None if st["state"] is None else st["state"].data_ptr(),
                                state_out_ptr=out[1].data_ptr(), ld_q=ld, ld_k=ld, ld_v=ld, ld_gates=2 * h)
    else:
        v, words = case["vocab"], case["words"]
        dev.beam_select_resident(st["logits"].data_ptr(), case["dtype"], case["groups"], case["beams"], v,
                                 st["scores"].data_ptr(), case["keep"], out[0].data_ptr(), out[1].data_ptr(),
                                 out[2].data_ptr(), last_ptr=st["last"].data_ptr(), eos=EOS, ld=v + case["pad"])
        dev.beam_gather_resident(st["states"].data_ptr(), out[3].data_ptr(), 4 * words, case["groups"], case["beams"],
                                 out[0].data_ptr(), case["keep"])
    return out


def _norm_sum(st):
    h = st["x"][:, :st["case"]["width"]].float()
    return h if st["residual"] is None else h + st["residual"][:, :st["case"]["width"]].float()


def _plain_norm(st):
    case, h = st["case"], _norm_sum(st)
    inv = 1.0 / torch.sqrt((h * h).mean(-1, keepdim=True) + 1e-5)
    out = [] if st["residual"] is None else [h.to(_type(case["dtype"]))]
    if case["op"] == "norm":
        return out + [(h * inv * st["gamma"]).to(_type(case["dtype"]))]
    # The inverse scales a whole row: codes go by h gamma alone.
    t = h * st["gamma"]
    most = t.abs().amax(-1, keepdim=True)
    codes = torch.where(most > 0, torch.round(t * (127.0 / most)), 0.0)
    y = torch.matmul(codes, st["w"].float().T) * (most / 127.0 * inv) * st["w_scales"]
    return out + [y.to(_type(case["out"]))]


def _plain_i8(st):
    case, k = st["case"], st["case"]["k"]
    y = torch.matmul(st["x"][:, :k].float(), st["w"][:, :k].float().T)
    return (y * st["x_scales"][:, None] * st["w_scales"]).to(_type(case["out"]))


def _delta_heads(case, row):
    """Queries, keys and values [tokens, heads, width] of the token rows, queries and keys for every head."""
    h, hk, dk, dv, n = case["heads"], case["key_heads"], case["d_key"], case["d_val"], row.shape[0]
    q, k = (row[:, i * hk * dk:(i + 1) * hk * dk].view(n, hk, dk).repeat_interleave(h // hk, 1) for i in (0, 1))
    return q, k, row[:, 2 * hk * dk:].view(n, h, dv)


def _bt(a):
    return a.transpose(-1, -2).contiguous()


def _plain_delta(st):
    """Chunks of 64 tokens: (1 + A) U = beta V - beta gamma K S, with A the decayed products of the keys before."""
    case, lens, h, dk = st["case"], st["lens_gpu"], st["case"]["heads"], st["case"]["d_key"]
    n, longest = len(st["lens"]), max(st["lens"])
    c = min(64, longest)
    chunks = -(-longest // c)
    t = torch.arange(chunks * c, device="cuda")
    live = t < lens[:, None]  # [n, T]
    at = ((lens.cumsum(0) - lens)[:, None] + t).clamp_max(st["row"].shape[0] - 1)

    def tiles(x):  # [tokens, heads, w] -> [n, heads, chunks, c, w], zeros behind a sequence's end
        x = torch.where(live[..., None, None], x.float()[at], 0.0)
        return x.view(n, chunks, c, h, -1).permute(0, 3, 1, 2, 4).contiguous()

    q, k, v = (tiles(x) for x in _delta_heads(case, st["row"]))
    g, beta = (tiles(st["gates"][:, i * h:(i + 1) * h, None])[..., 0] for i in (0, 1))
    total = g.double().cumsum(-1)
    i = torch.arange(c, device="cuda")
    decay = torch.where(i[:, None] >= i, torch.exp((total[..., :, None] - total[..., None, :]).clamp_max(0)), 0.0).float()
    gamma, rest = torch.exp(total).float()[..., None], torch.exp(total[..., -1:] - total).float()[..., None]
    a = torch.where(i[:, None] > i, beta[..., None] * decay * torch.matmul(k, _bt(k)), 0.0).double()
    inv, power = torch.eye(c, device="cuda", dtype=torch.float64) - a, a
    for _ in range(max(0, (c - 1).bit_length() - 1)):  # (1 + A)^-1 = (1 - A)(1 + A^2)(1 + A^4) ...
        power = torch.matmul(power, power)
        inv = inv + torch.matmul(inv, power)
    inv = inv.float()
    u0, w = torch.matmul(inv, beta[..., None] * v), torch.matmul(inv, beta[..., None] * gamma * k)
    kt = _bt(k * rest)
    # A chunk takes S to M S + B; composed over the chunks before it, doubling the span each time.
    m = gamma[..., -1:, :] * torch.eye(dk, device="cuda") - torch.matmul(kt, w)
    b = torch.matmul(kt, u0)
    if st["state"] is not None:
        b[:, :, 0] += torch.matmul(m[:, :, 0], st["state"])
    span = 1
    while span < chunks:
        b = torch.cat([b[:, :, :span], b[:, :, span:] + torch.matmul(m[:, :, span:], b[:, :, :-span])], 2)
        m = torch.cat([m[:, :, :span], torch.matmul(m[:, :, span:], m[:, :, :-span])], 2)
        span *= 2
    first = torch.zeros_like(b[:, :, 0]) if st["state"] is None else st["state"]
    entry = torch.cat([first[:, :, None], b[:, :, :-1]], 2)
    u = u0 - torch.matmul(w, entry)
    out = torch.matmul(torch.matmul(q, _bt(k)).mul_(decay), u) + gamma * torch.matmul(q, entry)
    out = out.permute(0, 2, 3, 1, 4).reshape(n, chunks * c, h, -1)[live] * st["scale"]
    # Tokens behind a sequence's end left the state as it is: their gates are 0.
    return [out.to(_type(case["dtype"])), b[:, :, -1].contiguous()]


def _plain_beam(st):
    case, v, keep = st["case"], st["case"]["vocab"], st["case"]["keep"]
    g, n = case["groups"], case["beams"]
    raw = st["logits"][:, :v].float()
    # In a beam by logit, then by id: one whole number for both, distinct for every token.
    bits = (raw + 0.0).view(torch.int32)
    ids = torch.arange(v, device="cuda")
    order = (bits ^ ((bits >> 31) & 0x7FFFFFFF)).long() * 2 ** 32 + (2 ** 32 - 1 - ids)
    few = min(keep, v)
    ids = 2 ** 32 - 1 - (order.topk(few, dim=-1).values & (2 ** 32 - 1))
    most = raw.amax(-1, keepdim=True).double()
    total = torch.log(torch.exp(raw.double() - most).sum(-1, keepdim=True)) + most
    cand = st["scores"].double()[..., None] + (raw.gather(1, ids).double() - total).view(g, n, few)
    # An ended beam stays as it is.
    ended = st["last"] == EOS
    only = torch.full_like(cand, -math.inf)
    only[..., 0] = st["scores"].double()
    cand = torch.where(ended[..., None], only, cand).view(g, n * few)
    ids = torch.where(ended[..., None], EOS, ids.view(g, n, few)).view(g, n * few)
    best, at = cand.sort(dim=-1, descending=True, stable=True)
    best, at = best[:, :keep], at[:, :keep]
    parents = torch.where(best > -math.inf, at // few, -1).to(torch.int32)
    tokens = torch.where(best > -math.inf, ids.gather(1, at), -1).to(torch.int32)
    rows = (torch.arange(g, device="cuda")[:, None] * n + parents).view(-1)
    return [parents, tokens, best.float(), st["states"][rows]]


_PLAIN = {"norm": _plain_norm, "norm_i8": _plain_norm, "i8": _plain_i8, "delta": _plain_delta, "beam": _plain_beam}


# ---------------------------------------------------------------------------
# What a pass cannot do without.


def work(case):
    if case["op"] in ("norm", "norm_i8"):
        n, d, size = case["rows"], case["width"], 4 if case["dtype"] == "f32" else 2
        rows = n * d * size * (3 if case["residual"] else 1)
        if case["op"] == "norm":
            return {"bytes": float(rows + n * d * size + 4 * d), "flops": 6.0 * n * d}
        out = 4 if case["out"] == "f32" else 2
        return {"bytes": float(rows + 4 * d + case["n"] * (d + 4) + n * case["n"] * out),
                "flops": 2.0 * n * d * case["n"] + 7.0 * n * d}
    if case["op"] == "i8":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": float(m * k + n * k + 4 * (m + n) + m * n * (4 if case["out"] == "f32" else 2)),
                "flops": 2.0 * m * n * k}
    if case["op"] == "delta":
        lens, h, hk, dk, dv = _lens(case), case["heads"], case["key_heads"], case["d_key"], case["d_val"]
        n, state, size = sum(lens), len(lens) * h * dk * dv * 4, 4 if case["dtype"] == "f32" else 2
        # The recurrence itself: decay, k S, the update and q S.
        return {"bytes": float(n * (2 * hk * dk + 2 * h * dv) * size + 8 * n * h + state * (2 if case["state"] else 1)),
                "flops": 7.0 * n * h * dk * dv}
    n, v, kept = case["groups"] * case["beams"], case["vocab"], case["groups"] * case["keep"]
    size = 4 if case["dtype"] == "f32" else 2
    return {"bytes": float(n * (v * size + 8) + 12 * kept + 4 * case["words"] * (min(n, kept) + kept)), "flops": 4.0 * n * v}


# ---------------------------------------------------------------------------
# The definitions in 64 bits.


def exact(case, seed):
    t = _INPUTS[case["op"]](case, seed)
    return {"norm": _exact_norm, "norm_i8": _exact_norm, "i8": _exact_i8, "delta": _exact_delta,
            "beam": _exact_beam}[case["op"]](case, t)


def _exact_product(x, w):
    """x w^T of whole numbers in 64 bits, some columns at a time."""
    block = max(1, (1 << 27) // w.shape[1])
    return torch.cat([torch.nn.functional.linear(x.double(), w[i:i + block].double())
                      for i in range(0, w.shape[0], block)], 1)


def _exact_norm(case, t):
    d = case["width"]
    h = t["x"][:, :d].double()
    if case["residual"]:
        h = h + t["residual"][:, :d].double()
    inv = (h.square().sum(-1, keepdim=True) / d + 1e-5).rsqrt()
    out = [h] if case["residual"] else []
    if case["op"] == "norm":
        return out + [inv * h * t["gamma"].double()]
    # The codes are whole numbers, given by their formula in 32 bits.
    v = h.float() * t["gamma"]
    peak = v.abs().max(-1, keepdim=True).values
    codes = (v * (torch.full_like(peak, 127.0) / peak)).round()
    scale = peak.double() * inv / 127.0
    return out + [_exact_product(codes, t["w"]) * scale * t["w_scales"].double()]


def _exact_i8(case, t):
    k = case["k"]
    return _exact_product(t["x"][:, :k], t["w"][:, :k]) * t["x_scales"].double()[:, None] * t["w_scales"].double()


def _exact_delta(case, t):
    """The recurrence, token by token: S = a S; S += k (beta (v - S^T k))^T; o = scale S^T q."""
    lens, h, n = torch.tensor(_lens(case), device="cuda"), case["heads"], len(_lens(case))
    q, k, v = (x.double() for x in _delta_heads(case, t["row"]))
    a, beta = t["gates"][:, :h].double().exp(), t["gates"][:, h:].double()
    s = torch.zeros(n, h, case["d_key"], case["d_val"], dtype=torch.float64, device="cuda")
    if t["state"] is not None:
        s += t["state"]
    out, first = torch.zeros_like(v), lens.cumsum(0) - lens
    order = torch.argsort(lens, descending=True)  # the longest first: those still running are a prefix
    s, first, sizes = s[order].clone(), first[order], sorted(_lens(case), reverse=True)
    for i in range(sizes[0]):
        while sizes[-1] <= i:
            sizes.pop()
        r = len(sizes)
        at = first[:r] + i
        s[:r].mul_(a[at][..., None, None])
        seen = (k[at][..., None] * s[:r]).sum(-2)
        s[:r].add_(k[at][..., None] * (beta[at][..., None] * (v[at] - seen))[..., None, :])
        out[at] = (q[at][..., None] * s[:r]).sum(-2) * t["scale"]
    return [out, s[torch.argsort(order)]]


def _exact_beam(case, t):
    g, n, v, keep = case["groups"], case["beams"], case["vocab"], case["keep"]
    scores = []
    for i in range(g):
        lp = torch.log_softmax(t["logits"][i * n:(i + 1) * n, :v].double(), -1) + t["scores"][i].double()[:, None]
        ended = t["last"][i] == EOS
        lp[ended] = -math.inf
        lp[ended, EOS] = t["scores"][i].double()[ended]
        scores.append(lp.flatten().sort(descending=True).values[:keep].clone())
    return [None, None, torch.stack(scores), None]
