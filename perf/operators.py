"""What the operators of a cache in 4 bits are timed and held to: appending to it, attending over it, and the log
probabilities by which a user sees what the 4 bits cost.

* ``append``: a layer's projected rows [q | k | v] get their head norms and rotation, the queries stay in the rows and keys and
  values go into pages in 4 bits.  Comes back: the queries, and the keys and values that the cache now holds for these rows
  (read from it), as the values they stand for.
* ``attend``: rows at given positions attend causally over their sequences' pages: single tokens, short runs that go on, whole
  prompts.  Comes back: the rows' results.
* ``logprobs``: the log probability of a given token in every row of logits, the row's entropy and its likeliest tokens.

The format: 16 neighbouring elements of a head are a group with one scale s, whose byte holds the upper bits of a half (5 of the
exponent, 3 of the fraction, no sign) that is s / 8; an element is a whole number c of [-7, 7] in 4 bits, held as c + 8, the even
element of a pair in the low half of its byte; the value is c s.  s is the group's largest magnitude over 7, rounded to the nearest
such number (at most 480), c the nearest whole number to x / s.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEVICE = "cuda:0"
DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}
PAGE = 64
GROUP = 16
UNIT = 8.0                 # a scale over the half that its byte is the upper part of
LARGEST_SCALE = 480.0


def _append(name, dtype, nq, nkv, d, past, new, norms=True, rotary=None, theta=1e6):
    return {"name": name, "op": "append", "dtype": dtype, "nq": nq, "nkv": nkv, "d": d, "past": past, "new": new, "norms": norms,
            "rotary": d if rotary is None else rotary, "theta": theta}


def _attend(name, dtype, nq, nkv, d, sequences, shortest, longest, new_least, new_most, window=0, lengths=0):
    return {"name": name, "op": "attend", "dtype": dtype, "nq": nq, "nkv": nkv, "d": d, "sequences": sequences, "shortest": shortest,
            "longest": longest, "new_least": new_least, "new_most": new_most, "window": window, "lengths": lengths}


def _logprobs(name, dtype, rows, vocab, top, masked=0.0):
    return {"name": name, "op": "logprobs", "dtype": dtype, "rows": rows, "vocab": vocab, "top": top, "masked": masked}


def listed():
    return [
        # one layer of a decoding step, eight sequences in the middle of their answers (the 1.7B decoder's heads)
        _append("append_8_tokens", "bfloat16", 16, 8, 128, "4000,17,1023,2500,64,3500,999,4095", "1,1,1,1,1,1,1,1"),
        # one layer of a prompt of 2,048 tokens, the benchmark's prompt
        _append("append_prompt_2048", "bfloat16", 16, 8, 128, "0", "2048"),
        # the 32-bit path, heads rotated in part and without norms, three sequences that go on by unequal runs
        _append("append_ragged_f32", "float32", 10, 2, 80, "700,0,63", "1,130,517", norms=False, rotary=40, theta=1e4),
        # the smallest step: one sequence early in its answer
        _attend("attend_1_at_900", "bfloat16", 16, 8, 128, 1, 900, 900, 1, 1),
        # the benchmark's decoding step: eight sequences of 4,096 tokens
        _attend("attend_8_at_4096", "bfloat16", 16, 8, 128, 8, 4096, 4096, 1, 1),
        # a server's step: 64 sequences of very unequal lengths (the 14B decoder's heads)
        _attend("attend_64_ragged", "bfloat16", 40, 8, 128, 64, 128, 8192, 1, 1, lengths=5),
        # two sequences as long as the decoders' configuration allows
        _attend("attend_2_at_40960", "bfloat16", 16, 8, 128, 2, 40960, 40960, 1, 1),
        # the benchmark's prompt attends to itself
        _attend("attend_prompt_2048", "bfloat16", 16, 8, 128, 1, 2048, 2048, 2048, 2048),
        # chats that go on by a few tokens over a window of keys
        _attend("attend_runs_window", "bfloat16", 40, 8, 128, 4, 5000, 7000, 5, 24, window=4096, lengths=3),
        # the 32-bit path's single tokens
        _attend("attend_f32", "float32", 12, 4, 64, 5, 40, 1500, 1, 1, lengths=2),
        # a decoding step that answers with the twenty likeliest tokens
        _logprobs("logprobs_8_top20", "float32", 8, 151936, 20),
        # a text of a thousand tokens is scored
        _logprobs("logprobs_1000_top5", "float32", 1000, 151936, 5),
    ]


def _between(rng, low, high):
    """A whole number whose logarithm is spread evenly."""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _drawn(rng):
    op = rng.choice(["append", "attend", "attend", "logprobs"])
    if op == "logprobs":
        vocab = _between(rng, 500, 152000)
        most = min(1000, max(1, int(1.2e8 / vocab)))
        return _logprobs("", rng.choice(["float32", "float32", "bfloat16"]), _between(rng, 1, most), vocab,
                         rng.choice([0, 1, 5, 20, 32]), rng.choice([0.0, 0.0, 0.4]))
    dtype = rng.choice(["bfloat16", "bfloat16", "bfloat16", "float32"])
    nkv = rng.choice([1, 2, 4, 8])
    nq = nkv * rng.choice([1, 2, 3, 4, 5, 8])
    if op == "append":
        d = rng.choice([64, 128]) if dtype == "bfloat16" else rng.choice([32, 64, 80, 128])
        count = _between(rng, 1, 32)
        tokens = _between(rng, 1, 60) if rng.random() < 0.5 else 1
        new = [rng.randint(1, tokens) for _ in range(count)]
        past = [_between(rng, 1, 8000) - 1 for _ in range(count)]
        return _append("", dtype, nq, nkv, d, ",".join(map(str, past)), ",".join(map(str, new)), norms=rng.random() < 0.7,
                       rotary=rng.choice([d, d, d // 2]), theta=rng.choice([1e4, 1e6]))
    if dtype == "float32":
        d = rng.choice([32, 64, 80, 128])
        longest = _between(rng, 1, 1500)
        return _attend("", dtype, nq, nkv, d, _between(rng, 1, 6), max(1, longest // rng.randint(1, 8)), longest, 1,
                       rng.choice([1, 1, 9]), window=rng.choice([0, 0, 200]), lengths=rng.randint(0, 999))
    d = rng.choice([64, 128, 128])
    kind = rng.choice(["decode", "decode", "runs", "prompt"])
    if kind == "prompt":
        longest = _between(rng, 50, 2000)
        return _attend("", dtype, nq, nkv, d, 1, longest, longest, longest, longest, window=rng.choice([0, 0, 500]))
    sequences = _between(rng, 1, 64)
    longest = _between(rng, 1, min(40960, 250000 // sequences))
    most = 1 if kind == "decode" else _between(rng, 2, 100)
    return _attend("", dtype, nq, nkv, d, sequences, max(1, longest // rng.choice([1, 3, 20])), longest, 1, most,
                   window=rng.choice([0, 0, 0, 1000]), lengths=rng.randint(0, 999))


def draw(rng: random.Random):
    case = _drawn(rng)
    while case["op"] == "attend" and work(case)["flops"] > 1.7e10:                       # as much as the listed prompt, at most
        case["longest"] = max(1, case["longest"] * 2 // 3)
        for key in ("shortest", "new_least", "new_most"):
            case[key] = min(case[key], case["longest"])
    return case


def _lengths(case):
    """(keys a sequence holds with its new tokens, new tokens) of every sequence: a seed of the case, so that every pass does the same work."""
    rng = random.Random(case["lengths"])
    keys = [_between(rng, case["shortest"], case["longest"]) for _ in range(case["sequences"])]
    if len(keys) > 1:
        keys[-1] = case["longest"]
    new = [min(k, rng.randint(case["new_least"], case["new_most"])) for k in keys]
    return keys, new


def _numbers(text):
    return [int(v) for v in text.split(",")]


# ---- the format ----------------------------------------------------------------------------------------------------

def _rounded_scale(s):
    """The nearest number of 4 significant bits (below 2^-11: the nearest multiple of 2^-14), ties to even."""
    step = torch.exp2(torch.floor(torch.log2(s.clamp(min=2.0 ** -11))) - 3.0)
    return torch.round(s / step) * step


def _quantised(x):
    """(codes [..., d], scales [..., d / 16]) of 32-bit x [..., d]; in 64 bits, since elements of 16 bits often lie right between two codes."""
    groups = x.double().unflatten(-1, (-1, GROUP))
    scale = _rounded_scale((groups.abs().amax(-1) / 7.0).clamp(max=LARGEST_SCALE))
    codes = torch.round(groups / torch.where(scale > 0, scale, 1.0)[..., None]).clamp(-7, 7)
    return codes.flatten(-2), scale


def _packed(codes, scale):
    """The bytes of codes and scales."""
    u = (codes + 8).to(torch.uint8)
    return u[..., 0::2] | (u[..., 1::2] << 4), ((scale / UNIT).to(torch.float16).view(torch.int16) >> 7).to(torch.uint8)


def _unpacked(codes, scales):
    """The values of bytes, in 32 bits."""
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).to(torch.float32) - 8.0
    s = (scales.to(torch.int16) << 7).view(torch.float16).to(torch.float32) * UNIT
    return (c.unflatten(-1, (-1, GROUP)) * s[..., None]).flatten(-2)


# ---- inputs --------------------------------------------------------------------------------------------------------

def _table(sequences, pages_each, gen):
    """A page table [sequences, most pages] whose pages lie in no order, as after a while of serving."""
    most = max(pages_each)
    order = torch.randperm(sum(pages_each), device=DEVICE, generator=gen).to(torch.int32)
    table = torch.zeros((sequences, most), dtype=torch.int32, device=DEVICE)
    at = 0
    for s, n in enumerate(pages_each):
        table[s, :n] = order[at:at + n]
        at += n
    return table


def _step(past, new):
    """The device's and the host's lists of a step's rows."""
    slot = [s for s, n in enumerate(new) for _ in range(n)]
    pos = [p + i for p, n in zip(past, new) for i in range(n)]
    start = [0]
    for n in new:
        start.append(start[-1] + n)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=DEVICE)
    return {"row_slot": ints(slot), "row_pos": ints(pos), "seq_start": ints(start), "seq_slot": ints(list(range(len(new)))),
            "seq_past": ints(past), "tokens": ints([0] * len(slot)), "want": ints([]), "past": past, "new": new}


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    normal = lambda *shape: torch.randn(*shape, device=DEVICE, generator=gen)
    state = {"case": dict(case)}
    if case["op"] == "logprobs":
        rows, vocab = case["rows"], case["vocab"]
        logits = normal(rows, vocab) * 2.5
        likely = torch.randint(0, vocab, (rows, 8), device=DEVICE, generator=gen)        # a few tokens that the model finds likely
        logits.scatter_add_(1, likely, 8.0 + 3.0 * normal(rows, 8))
        tokens = likely[:, 0].clone()
        rare = torch.rand(rows, device=DEVICE, generator=gen) < 0.3
        tokens[rare] = torch.randint(0, vocab, (rows,), device=DEVICE, generator=gen)[rare]
        if case["masked"]:                                                               # a grammar forbids some of the tokens
            gone = torch.rand(rows, vocab, device=DEVICE, generator=gen) < case["masked"]
            gone.scatter_(1, tokens[:, None], False)
            logits.masked_fill_(gone, -math.inf)
        return state | {"logits": logits.to(DTYPES[case["dtype"]]), "tokens": tokens.to(torch.int32)}
    nq, nkv, d = case["nq"], case["nkv"], case["d"]
    dtype = DTYPES[case["dtype"]]
    if case["op"] == "append":
        past, new = _numbers(case["past"]), _numbers(case["new"])
        pages = [(p + n + PAGE - 1) // PAGE for p, n in zip(past, new)]
        spread = torch.exp(0.5 * normal((nq + 2 * nkv) * d))                             # channels differ, as a model's do
        state["qkv"] = (normal(sum(new), (nq + 2 * nkv) * d) * spread).to(dtype)
        state["q_out"] = torch.empty((sum(new), nq * d), dtype=dtype, device=DEVICE)
        state["q_gain"], state["k_gain"] = ((1.0 + 0.3 * normal(d)).to(dtype) if case["norms"] else None for _ in range(2))
        half = case["rotary"] // 2
        state["inv_freq"] = torch.pow(torch.tensor(case["theta"], dtype=torch.float64),
                                      -torch.arange(half, dtype=torch.float64) / half).to(torch.float32).to(DEVICE)
        state["eps"] = 1e-6
        shape = (sum(pages), nkv, PAGE)
        state["codes"] = [torch.zeros(shape + (d // 2,), dtype=torch.uint8, device=DEVICE) for _ in range(2)]
        state["scales"] = [torch.zeros(shape + (d // GROUP,), dtype=torch.uint8, device=DEVICE) for _ in range(2)]
    else:
        keys, new = _lengths(case)
        past = [k - n for k, n in zip(keys, new)]
        pages = [(k + PAGE - 1) // PAGE for k in keys]
        state["qkv"] = (1.5 * normal(sum(new), (nq + 2 * nkv) * d)).to(dtype)
        state["out"] = torch.empty((sum(new), nq * d), dtype=dtype, device=DEVICE)
        state["codes"], state["scales"] = [], []
        for is_key in (True, False):
            offset = 0.5 * normal(nkv, 1, d) if is_key else torch.zeros(nkv, 1, d, device=DEVICE)    # keys' channels have means
            codes, scales = [], []
            for at in range(0, sum(pages), 512):
                n = min(512, sum(pages) - at)
                c, s = _packed(*_quantised(normal(n, nkv, PAGE, d) + offset))
                codes.append(c)
                scales.append(s)
            state["codes"].append(torch.cat(codes))
            state["scales"].append(torch.cat(scales))
    state["table"] = _table(len(new), pages, gen)
    return state | _step(past, new)


# ---- the plain forms -----------------------------------------------------------------------------------------------

def _plain_rotated(x, pos, inv_freq):
    """x [rows, heads, d] with pairs (i, i + rotated / 2) turned by pos * inv_freq."""
    half = inv_freq.numel()
    angle = pos.double()[:, None] * inv_freq.double()
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    a, b = x[..., :half], x[..., half:2 * half]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., 2 * half:]], -1)


def _plain_append(st):
    case = st["case"]
    nq, nkv, d = case["nq"], case["nkv"], case["d"]
    x = st["qkv"].float().unflatten(-1, (nq + 2 * nkv, d))
    q, k, v = x[:, :nq], x[:, nq:nq + nkv], x[:, nq + nkv:]
    if case["norms"]:
        q = q / torch.sqrt((q * q).mean(-1, keepdim=True) + st["eps"]) * st["q_gain"].float()
        k = k / torch.sqrt((k * k).mean(-1, keepdim=True) + st["eps"]) * st["k_gain"].float()
    q, k = _plain_rotated(q, st["row_pos"], st["inv_freq"]), _plain_rotated(k, st["row_pos"], st["inv_freq"])
    page = st["table"][st["row_slot"].long(), st["row_pos"].long() // PAGE].long()
    place = st["row_pos"].long() % PAGE
    values = []
    for i, y in enumerate((k, v)):
        codes, scales = _packed(*_quantised(y))
        st["codes"][i][page, :, place] = codes
        st["scales"][i][page, :, place] = scales
        values.append(_unpacked(st["codes"][i][page, :, place], st["scales"][i][page, :, place]).to(torch.bfloat16))
    return {"q": q.flatten(1).to(st["qkv"].dtype), "keys": values[0], "values": values[1]}


def _plain_attend(st):
    case = st["case"]
    nq, nkv, d, window = case["nq"], case["nkv"], case["d"], case["window"]
    start, past = st["seq_start"].long(), st["seq_past"].long()
    B, most = len(st["new"]), max(st["new"])
    row = start[:-1, None] + torch.arange(most, device=DEVICE)                           # [sequence, new token] -> row
    real = row < start[1:, None]
    q = st["qkv"][:, :nq * d].float()[row.clamp(max=int(st["qkv"].shape[0]) - 1)]        # [B, new, nq d]
    q = q.unflatten(-1, (nkv, nq // nkv, d)).permute(0, 2, 3, 1, 4).flatten(2, 3)        # [B, nkv, group new, d]
    k, v = (_unpacked(c[st["table"].long()], s[st["table"].long()]).transpose(1, 2).flatten(2, 3)
            for c, s in zip(st["codes"], st["scales"]))                                  # [B, nkv, keys, d]
    pos = past[:, None] + torch.arange(most, device=DEVICE)                              # [B, new]
    at = torch.arange(k.shape[2], device=DEVICE)
    seen = at <= pos[..., None]
    if window:
        seen &= at > pos[..., None] - window
    scores = (q @ k.transpose(2, 3) / math.sqrt(d)).unflatten(2, (nq // nkv, most))
    scores = torch.where(seen[:, None, None], scores, -math.inf)
    weights = torch.exp(scores - scores.amax(-1, keepdim=True))
    weights = (weights / weights.sum(-1, keepdim=True)).flatten(2, 3)
    out = (weights @ v).unflatten(2, (nq // nkv, most)).permute(0, 3, 1, 2, 4).flatten(2)      # [B, new, nq d]
    return out[real].to(st["qkv"].dtype)


def _plain_logprobs(st):
    x = st["logits"].float()
    x = torch.where(torch.isfinite(x), x, -math.inf)
    most = x.amax(-1, keepdim=True)
    e = torch.exp(x - most)
    total = e.sum(-1, keepdim=True)
    norm = most + torch.log(total)
    found = {"logprobs": (x.gather(1, st["tokens"].long()[:, None]) - norm)[:, 0],
             "entropy": (torch.log(total) - (e * torch.where(e > 0, x - most, 0.0)).sum(-1, keepdim=True) / total)[:, 0]}
    if st["case"]["top"]:
        value, index = torch.sort(x, dim=-1, descending=True, stable=True)
        value, index = value[:, :st["case"]["top"]], index[:, :st["case"]["top"]]
        found["top_ids"] = torch.where(torch.isfinite(value), index, -1).to(torch.int32)
        found["top_logprobs"] = value - norm
    return found


def run(state):
    op = state["case"]["op"]
    if not own:
        return {"append": _plain_append, "attend": _plain_attend, "logprobs": _plain_logprobs}[op](state)
    import citlali_b200 as cb
    from citlali_b200 import ops
    case = state["case"]
    if op == "logprobs":
        return ops.token_logprobs(state["logits"], state["tokens"], top=case["top"])
    kv = cb.KVView(cb.Packed4(state["codes"][0], state["scales"][0]), cb.Packed4(state["codes"][1], state["scales"][1]), state["table"], PAGE,
                   cb.KVRequirement(case["nkv"], case["d"], case.get("window") or None, packed4=True))
    if op == "append":
        ops.cache4_append(state["qkv"], kv, state["row_slot"], state["row_pos"], case["nq"], case["nkv"], case["d"], state["inv_freq"],
                          case["rotary"], state["q_gain"], state["k_gain"], state["eps"], q_out=state["q_out"])
        keys, values = ops.cache4_read(kv, state["row_slot"], state["row_pos"])
        return {"q": state["q_out"], "keys": keys, "values": values}
    batch = cb.StepBatch(state["tokens"], state["row_slot"], state["row_pos"], state["seq_start"], state["seq_slot"], state["seq_past"],
                         state["want"], slots=list(range(len(state["new"]))), past=state["past"], n_new=state["new"])
    ops.cache4_attention(state["qkv"], state["qkv"].shape[1], kv, batch, state["out"], case["nq"], case["nkv"], case["d"],
                         case["window"], 1.0 / math.sqrt(case["d"]))
    return state["out"]


# ---- 64 bits -------------------------------------------------------------------------------------------------------

def _exact_values(x):
    """What x (float64) is held as: by the table of all the scales there are."""
    bits = torch.arange(0, 0x5381, 0x80, dtype=torch.int16).view(torch.float16).double().to(x.device) * 8
    shape = x.shape
    x = x.reshape(-1, GROUP)
    wanted = torch.clamp(x.abs().max(dim=1).values / 7.0, max=LARGEST_SCALE)
    above = torch.searchsorted(bits, wanted).clamp(max=bits.numel() - 1)
    below = (above - 1).clamp(min=0)
    up, down = (bits[above] - wanted).abs(), (wanted - bits[below]).abs()
    pick = torch.where((up < down) | ((up == down) & (above % 2 == 0)), above, below)
    s = bits[pick][:, None]
    c = torch.where(s > 0, torch.round(x / s.clamp(min=1e-30)), torch.zeros_like(x))
    return (c.clamp(-7, 7) * s).reshape(shape)


def _exact_cached(state, i, sequence, keys):
    """Keys (i = 0) or values (1) of a sequence in float64 [nkv, keys, d], page by page as the table names them."""
    pages = state["table"][sequence, :(keys + PAGE - 1) // PAGE].long()
    code = state["codes"][i][pages].to(torch.int64)
    value = torch.empty(code.shape[:-1] + (2 * code.shape[-1],), dtype=torch.float64, device=DEVICE)
    value[..., 0::2] = (code % 16 - 8).double()
    value[..., 1::2] = (code // 16 - 8).double()
    b = state["scales"][i][pages].to(torch.int64)
    e, f = b // 8, (b % 8).double()
    s = torch.where(e == 0, f * 2.0 ** -14, (1 + f / 8) * torch.exp2(e.double() - 12))
    value *= s.repeat_interleave(GROUP, dim=-1)
    return value.transpose(0, 1).flatten(1, 2)[:, :keys]


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "logprobs":
        x = st["logits"].double()
        x[~torch.isfinite(x)] = -math.inf
        p = torch.softmax(x, -1)
        log_p = torch.log_softmax(x, -1)
        rows = torch.arange(x.shape[0], device=DEVICE)
        found = {"logprobs": log_p[rows, st["tokens"].long()], "entropy": -torch.special.xlogy(p, p).sum(-1)}
        if case["top"]:
            ids, logs = [], []
            rest = x.clone()
            for _ in range(case["top"]):
                top = rest.max(-1, keepdim=True).values
                first = (rest == top).to(torch.uint8).argmax(-1)          # ties: the lowest index
                none = torch.isinf(top[:, 0])
                ids.append(torch.where(none, -1, first).to(torch.int32))
                logs.append(torch.where(none, -math.inf, log_p[rows, first]))
                rest[rows, first] = -math.inf
            found["top_ids"], found["top_logprobs"] = torch.stack(ids, -1), torch.stack(logs, -1)
        return found
    nq, nkv, d = case["nq"], case["nkv"], case["d"]
    if case["op"] == "append":
        heads = st["qkv"].double().reshape(-1, nq + 2 * nkv, d)
        done = []
        for at, n, gain in ((0, nq, st["q_gain"]), (nq, nkv, st["k_gain"])):
            y = heads[:, at:at + n]
            if gain is not None:
                y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + st["eps"]) * gain.double()
            turn = torch.polar(torch.ones((), dtype=torch.float64, device=DEVICE),
                               st["row_pos"].double()[:, None, None] * st["inv_freq"].double())
            half = case["rotary"] // 2
            z = torch.complex(y[..., :half].contiguous(), y[..., half:2 * half].contiguous()) * turn
            done.append(torch.cat([z.real, z.imag, y[..., 2 * half:]], -1))
        return {"q": done[0].reshape(-1, nq * d), "keys": _exact_values(done[1]), "values": _exact_values(heads[:, nq + nkv:])}
    out = torch.empty((sum(st["new"]), nq * d), dtype=torch.float64, device=DEVICE)
    row = 0
    for s, (past, n) in enumerate(zip(st["past"], st["new"])):
        k, v = _exact_cached(st, 0, s, past + n), _exact_cached(st, 1, s, past + n)
        far = torch.arange(past, past + n, device=DEVICE)[:, None] - torch.arange(past + n, device=DEVICE)[None]
        hidden = (far < 0) | (far >= case["window"]) if case["window"] else far < 0
        for h in range(nq):
            q = st["qkv"][row:row + n, h * d:(h + 1) * d].double()
            score = (q @ k[h // (nq // nkv)].T * d ** -0.5).masked_fill_(hidden, -math.inf)
            out[row:row + n, h * d:(h + 1) * d] = torch.softmax(score, -1) @ v[h // (nq // nkv)]
        row += n
    return out


def work(case):
    if case["op"] == "logprobs":
        size = torch.empty((), dtype=DTYPES[case["dtype"]]).element_size()
        entries = case["rows"] * case["vocab"]
        return {"bytes": entries * size + case["rows"] * (4 + 8 + 8 * case["top"]), "flops": 6 * entries}
    nq, nkv, d = case["nq"], case["nkv"], case["d"]
    size = torch.empty((), dtype=DTYPES[case["dtype"]]).element_size()
    held = nkv * (d // 2 + d // GROUP)                                   # bytes of a token's key, or of its value
    if case["op"] == "append":
        rows = sum(_numbers(case["new"]))
        # q, k, v in, q out, 4 bits out, and the values that the cache stands for
        return {"bytes": rows * ((2 * nq + 2 * nkv) * d * size + 2 * held + 2 * nkv * d * 2), "flops": rows * (nq + 2 * nkv) * d * 8}
    keys, new = _lengths(case)
    window = case["window"] or 1 << 30
    seen = sum(min(window, k - n + i + 1) for k, n in zip(keys, new) for i in range(n))
    read = sum(min(k, window + n - 1) for k, n in zip(keys, new))
    return {"bytes": 2 * read * held + 2 * sum(new) * nq * d * size, "flops": 4 * seen * nq * d}
