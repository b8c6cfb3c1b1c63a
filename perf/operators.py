"""Cases of the text decoder's operators: the 4-bit paged key/value cache
(written and read back), the attention over it, and token sampling.

Where `own` is false, run() computes the operators in plain torch operations
in 32 bits; where it is true, through ppocr_b200.decode."""

import math
import sys
from pathlib import Path

import torch

own = False

GROUP = 32  # channels that share a scale and a minimum
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
LIMIT = {"fp16": 65000.0, "bf16": 2.0 ** 126}  # finite values saturate here


def listed():
    return [
        # One token for each of 16 lines being decoded: launch latency.
        {"name": "append_step", "op": "append", "batch": 16, "new_lo": 1, "new_hi": 1, "past": 211,
         "heads": 8, "kv_heads": 4, "dim": 64, "page": 32, "type": "fp16"},
        # Page prompts (visual tokens) of very different lengths, long ones among them.
        {"name": "append_prompts", "op": "append", "batch": 24, "new_lo": 37, "new_hi": 5001, "past": 0,
         "heads": 16, "kv_heads": 8, "dim": 128, "page": 64, "type": "bf16"},
        # One line, one token, every head with its own cache head: the smallest call.
        {"name": "step_line", "op": "attend", "batch": 1, "new_lo": 1, "new_hi": 1, "past": 76, "spread": 0,
         "heads": 8, "kv_heads": 8, "dim": 64, "page": 16, "window": 0, "sinks": 0, "type": "fp16"},
        # A serving batch in the middle of its answers, ragged.
        {"name": "step_batch", "op": "attend", "batch": 64, "new_lo": 1, "new_hi": 1, "past": 90, "spread": 2000,
         "heads": 16, "kv_heads": 4, "dim": 128, "page": 64, "window": 0, "sinks": 0, "type": "bf16"},
        # Whole documents in the cache: the step is the reading of the cache.
        {"name": "step_long", "op": "attend", "batch": 16, "new_lo": 1, "new_hi": 1, "past": 32000, "spread": 767,
         "heads": 32, "kv_heads": 8, "dim": 128, "page": 128, "window": 0, "sinks": 0, "type": "fp16"},
        # The same with a sliding window and four first tokens.
        {"name": "step_window", "op": "attend", "batch": 48, "new_lo": 1, "new_hi": 1, "past": 9000, "spread": 3001,
         "heads": 16, "kv_heads": 2, "dim": 64, "page": 32, "window": 2048, "sinks": 4, "type": "bf16"},
        # Prompts of line crops: many short ragged ones.
        {"name": "prompt_lines", "op": "attend", "batch": 48, "new_lo": 21, "new_hi": 300, "past": 0, "spread": 0,
         "heads": 8, "kv_heads": 8, "dim": 64, "page": 32, "window": 0, "sinks": 0, "type": "fp16"},
        # A page's prompt at once: the tensor cores bound it.
        {"name": "prompt_page", "op": "attend", "batch": 2, "new_lo": 4096, "new_hi": 4096, "past": 0, "spread": 0,
         "heads": 16, "kv_heads": 4, "dim": 128, "page": 64, "window": 0, "sinks": 0, "type": "bf16"},
        # A chunk of a long prompt, through a window, over what is already cached.
        {"name": "prompt_chunk", "op": "attend", "batch": 4, "new_lo": 500, "new_hi": 513, "past": 7000, "spread": 501,
         "heads": 16, "kv_heads": 4, "dim": 128, "page": 128, "window": 4096, "sinks": 8, "type": "fp16"},
        # The next token of a few lines, over the recognizer's vocabulary.
        {"name": "sample_lines", "op": "sample", "rows": 4, "vocab": 18385, "type": "fp16",
         "temperature": 0.8, "top_k": 50, "top_p": 0.95, "min_p": 0.0},
        # A serving batch over the same vocabulary, nucleus only.
        {"name": "sample_batch", "op": "sample", "rows": 256, "vocab": 18385, "type": "fp32",
         "temperature": 1.0, "top_k": 0, "top_p": 0.9, "min_p": 0.0},
        # A large vocabulary, all of it in the running before min-p.
        {"name": "sample_wide", "op": "sample", "rows": 96, "vocab": 131072, "type": "bf16",
         "temperature": 1.3, "top_k": 0, "top_p": 0.98, "min_p": 0.01},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "step", "step", "prompt", "prompt", "sample"])
    if op == "sample":
        rows, vocab = _log(rng, 1, 512), _log(rng, 1000, 150000)
        rows = max(1, min(rows, 96 * 131072 // vocab))
        return {"op": "sample", "rows": rows, "vocab": vocab, "type": rng.choice(["fp16", "bf16", "fp32"]),
                "temperature": rng.choice([0.0, 0.6, 0.8, 1.0, 1.3]), "top_k": rng.choice([0, 0, 1, 20, 50, 400]),
                "top_p": rng.choice([1.0, 0.98, 0.9, 0.5]), "min_p": rng.choice([0.0, 0.0, 0.02, 0.1])}
    dim = rng.choice([32, 64, 128])
    kv = rng.choice([1, 2, 4, 8])
    c = {"op": "append" if op == "append" else "attend", "heads": kv * rng.choice([1, 2, 4, 8]), "kv_heads": kv,
         "dim": dim, "page": rng.choice([16, 32, 64, 128]), "type": rng.choice(["fp16", "bf16"])}
    if op == "append":
        hi = _log(rng, 1, 5000)
        c |= {"new_hi": hi, "new_lo": rng.randint(1, hi), "past": rng.choice([0, _log(rng, 1, 3000)])}
        c["batch"] = _log(rng, 1, max(2, min(128, 500000 // (c["past"] + hi) // kv)))
        return c
    if op == "step":
        n = rng.choice([1, 1, 1, 2, 4])
        c |= {"new_lo": n, "new_hi": n, "past": _log(rng, 1, 30000)}
        c["spread"] = rng.choice([0, c["past"] // 2])
        c["batch"] = _log(rng, 1, max(2, min(128, 4000000 // ((c["past"] + c["spread"]) * kv))))
    else:
        hi = _log(rng, 8, 3000)
        c |= {"new_hi": hi, "new_lo": rng.randint(1, hi), "past": rng.choice([0, 0, _log(rng, 1, 6000)])}
        c["spread"] = rng.choice([0, c["past"] // 3])
        pairs = lambda: c["new_hi"] * (c["new_hi"] + c["past"] + c["spread"]) * c["heads"]  # noqa: E731
        while pairs() > 500_000_000:
            c["new_hi"] = c["new_hi"] * 2 // 3
        c["new_lo"] = min(c["new_lo"], c["new_hi"])
        c["batch"] = max(1, min(64, _log(rng, 1, max(2, 500_000_000 // pairs())), 500_000_000 // pairs()))
    c["window"] = rng.choice([0, 0, _log(rng, 16, 4096)])
    c["sinks"] = rng.choice([0, 4, 17]) if c["window"] else 0
    return c


def _spread(n, lo, hi, turn):
    """n whole numbers between lo and hi, the same ones for every seed."""
    return [lo + int(((i * 0.6180339887 + turn) % 1.0) * (hi - lo + 1)) for i in range(n)]


def _lengths(case):
    """(new tokens, length with them) of each sequence."""
    new = _spread(case["batch"], case["new_lo"], case["new_hi"], 0.9)
    past = _spread(case["batch"], case["past"], case["past"] + case.get("spread", 0), 0.4)
    return new, [a + b for a, b in zip(new, past)]


def work(case):
    if case["op"] == "sample":
        size = 4 if case["type"] == "fp32" else 2
        return {"bytes": case["rows"] * (case["vocab"] * size + 16 + 16), "flops": case["rows"] * case["vocab"] * 6}
    new, lengths = _lengths(case)
    d, kv, h = case["dim"], case["kv_heads"], case["heads"]
    held = d + d // GROUP * 8  # bytes of one token's keys and values in one head
    if case["op"] == "append":  # read and quantise, write, read, write back
        n = sum(new) * kv
        return {"bytes": n * (8 * d + 2 * held), "flops": n * 2 * d * 6}
    w, s = case["window"], case["sinks"]
    pairs = tokens = 0
    for n, length in zip(new, lengths):
        first = length - n
        if not w:
            pairs += n * first + n * (n + 1) // 2
            tokens += length
            continue
        for pos in range(first, length):
            low = max(0, pos + 1 - w)
            pairs += pos + 1 - low + min(s, low)
        low = max(0, first + 1 - w)
        tokens += length - low + min(s, low)
    return {"bytes": sum(new) * h * d * 4 + tokens * kv * held, "flops": 4 * d * h * pairs}


# ------------------------------------------------------------------- inputs
def _quantise(x, kind):
    """Codes (0..15, float) and the 16-bit scale and minimum of x's groups of 32 channels, in 32 bits."""
    x = torch.nan_to_num(x.float(), nan=0.0, posinf=LIMIT[kind], neginf=-LIMIT[kind]).clamp(-LIMIT[kind], LIMIT[kind])
    x = x.unflatten(-1, (-1, GROUP))
    low, high = x.amin(-1), x.amax(-1)
    low16 = low.to(DTYPES[kind])
    scale16 = ((high - low16.float()) / 15).to(DTYPES[kind])
    scale = scale16.float()[..., None]
    inv = torch.where(scale > 1e-30, 1 / scale, 0)
    codes = torch.clamp(torch.round((x - low16.float()[..., None]) * inv), 0, 15)
    return codes.flatten(-2), scale16, low16


def _views(state):
    """Key codes, value codes, key and value (scale, minimum) of the pool, by page, head and slot."""
    c, pool = state["case"], state["pool"]
    p, d, g = c["page"], c["dim"], c["dim"] // GROUP
    n, m = p * d // 2, p * g * 4
    codes = [pool[..., a:a + n].unflatten(-1, (p, d // 2)) for a in (0, n)]
    params = [pool[..., a:a + m].view(DTYPES[c["type"]]).unflatten(-1, (p, g, 2)) for a in (2 * n, 2 * n + m)]
    return codes + params


def _store(code_view, param_view, where, x, kind):
    codes, scale, low = _quantise(x, kind)
    codes = codes.to(torch.uint8)
    code_view[where] = codes[..., 0::2] | (codes[..., 1::2] << 4)
    param_view[where] = torch.stack([scale, low], -1)


def _load(code_view, param_view, where):
    codes, params = code_view[where], param_view[where].float()
    codes = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).float()
    return codes.unflatten(-1, (-1, GROUP)).mul(params[..., 0:1]).add(params[..., 1:2]).flatten(-2)


def prepare(case, seed):
    dev = torch.device("cuda")
    rng = torch.Generator(device=dev)
    rng.manual_seed(seed)
    if case["op"] == "sample":
        rows, vocab = case["rows"], case["vocab"]
        # Logits as a trained head gives them: a wide bulk and a few words far above it.
        logits = torch.randn(rows, vocab, device=dev, generator=rng) * 2.0
        top = torch.randint(0, vocab, (rows, 12), device=dev, generator=rng)
        logits.scatter_add_(1, top, 9.0 + 4.0 * torch.rand(rows, 12, device=dev, generator=rng))
        full = lambda v, t: torch.full((rows,), v, device=dev, dtype=t)  # noqa: E731
        return {"case": case, "logits": logits.to(DTYPES[case["type"]]),
                "uniform": torch.rand(rows, device=dev, generator=rng),
                "temperature": full(case["temperature"], torch.float32), "top_k": full(case["top_k"], torch.int32),
                "top_p": full(case["top_p"], torch.float32), "min_p": full(case["min_p"], torch.float32)}
    kind, d, kv, h, p = case["type"], case["dim"], case["kv_heads"], case["heads"], case["page"]
    new, lengths = _lengths(case)
    batch, tokens = case["batch"], sum(new)
    width = -(-max(lengths) // p)
    pages = batch * width
    block = p * (d + d // GROUP * 8)
    state = {"case": case, "pool": torch.zeros(pages, kv, block, dtype=torch.uint8, device=dev),
             "table": torch.randperm(pages, device=dev, generator=rng).to(torch.int32).view(batch, width),
             "lengths": torch.tensor(lengths, dtype=torch.int32, device=dev), "max_new": max(new)}
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    state["starts"] = torch.tensor(starts, dtype=torch.int32, device=dev)
    # Keys have a few channels much wider than the others.
    wide = torch.exp(0.5 * torch.randn(kv, d, device=dev, generator=rng))
    # One projection's output holds queries, keys and values of each token side by side.
    qkv = torch.randn(tokens, (h + 2 * kv) * d, device=dev, generator=rng)
    qkv[:, h * d:(h + kv) * d] *= wide.flatten()
    qkv = qkv.to(DTYPES[kind])
    state["q"] = qkv[:, :h * d].unflatten(-1, (h, d))
    state["k"] = qkv[:, h * d:(h + kv) * d].unflatten(-1, (kv, d))
    state["v"] = qkv[:, (h + kv) * d:].unflatten(-1, (kv, d))
    if case["op"] == "attend":
        views = _views(state)
        some = max(1, (1 << 26) // (kv * p * d))
        for a in range(0, pages, some):
            n = min(some, pages - a)
            where = slice(a, a + n)
            for x, codes, params in ((wide[:, None], views[0], views[2]), (1.0, views[1], views[3])):
                _store(codes, params, where, torch.randn(n, kv, p, d, device=dev, generator=rng) * x, kind)
    if own:  # the handle that a user's program keeps: the geometry, the pool and its workspace
        at = str(Path(__file__).resolve().parent.parent / "ppocrv6-native-server_b200")
        if at not in sys.path:
            sys.path.insert(0, at)
        from ppocr_b200 import decode

        state["cache"] = decode.KvCache4(pages, p, kv, d, dtype=DTYPES[kind], device="cuda:0", pool=state["pool"])
    return state


# ---------------------------------------------------------------- operators
def run(state):
    case = state["case"]
    if case["op"] == "sample":
        return _own_sample(state) if own else _plain_sample(state)
    if case["op"] == "append":
        return _own_append(state) if own else _plain_append(state)
    return _own_attend(state) if own else _plain_attend(state)


def _own_append(s):
    s["cache"].append(s["k"], s["v"], s["table"], s["lengths"], starts=s["starts"], max_new=s["max_new"])
    return s["cache"].read(s["table"], s["lengths"], s["k"].shape[0], starts=s["starts"], max_new=s["max_new"])


def _own_attend(s):
    c = s["case"]
    return s["cache"].attention(s["q"], s["table"], s["lengths"], starts=s["starts"], max_new=s["max_new"],
                                window=c["window"], sinks=c["sinks"])


def _own_sample(s):
    at = str(Path(__file__).resolve().parent.parent / "ppocrv6-native-server_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    from ppocr_b200 import decode

    return decode.sample(s["logits"], s["uniform"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
                         min_p=s["min_p"])


def _places(s):
    """Sequence and position of every new token."""
    starts, lengths = s["starts"].long(), s["lengths"].long()
    tokens = s["q"].shape[0]
    at = torch.arange(tokens, device=starts.device)
    seq = torch.searchsorted(starts, at, right=True) - 1
    return seq, lengths[seq] - (starts[seq + 1] - at)


def _plain_append(s):
    p, kind = s["case"]["page"], s["case"]["type"]
    seq, pos = _places(s)
    page = s["table"].long()[seq, pos // p]
    where = (page, slice(None), pos % p)
    kc, vc, kp, vp = _views(s)
    _store(kc, kp, where, s["k"], kind)
    _store(vc, vp, where, s["v"], kind)
    return _load(kc, kp, where).to(DTYPES[kind]), _load(vc, vp, where).to(DTYPES[kind])


def _plain_attend(s):
    c = s["case"]
    kv, d, kind = c["kv_heads"], c["dim"], c["type"]
    starts, lengths, table = s["starts"].long(), s["lengths"].long(), s["table"].long()
    kc, vc, kp, vp = _views(s)
    # [batch, kv heads, keys, dim], zero past each length
    key = torch.arange(table.shape[1] * c["page"], device=table.device)
    held = (key[None] < lengths[:, None])[:, None, :, None]
    k = torch.where(held, _load(kc, kp, table).transpose(1, 2).flatten(2, 3), 0)
    v = torch.where(held, _load(vc, vp, table).transpose(1, 2).flatten(2, 3), 0)
    # queries of each sequence, padded to the longest: [batch, kv heads, group * new, dim]
    n = starts[1:] - starts[:-1]
    i = torch.arange(s["max_new"], device=table.device)
    row = (starts[:-1, None] + i).clamp(max=s["q"].shape[0] - 1)
    q = s["q"].float()[row].unflatten(2, (kv, -1)).permute(0, 2, 3, 1, 4)
    group = q.shape[2]
    scores = (q.flatten(2, 3) @ k.transpose(2, 3)).mul_(1 / math.sqrt(d)).unflatten(2, (group, -1))
    pos = (lengths - n)[:, None] + i
    seen = key <= pos[..., None]
    if c["window"]:
        seen &= (key > pos[..., None] - c["window"]) | (key < c["sinks"])
    scores = scores.masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True).clamp(min=-3e38)
    e = scores.sub_(top).exp_()
    total = e.sum(-1, keepdim=True)
    o = (e.flatten(2, 3) @ v).unflatten(2, (group, -1)) / torch.where(total > 0, total, 1)
    o = o.permute(0, 3, 1, 2, 4).flatten(2, 3)
    return o[i[None] < n[:, None]].to(DTYPES[kind])


def _part(whole, share24):
    """floor(whole * share24 / 2^24) in 64-bit whole numbers, where the product itself may not fit."""
    return share24 * (whole >> 24) + (share24 * (whole & 0xFFFFFF) >> 24)


def _plain_sample(s):
    x = s["logits"].float()
    vocab = x.shape[1]
    x = torch.where(torch.isnan(x), -math.inf, x)
    greedy = ~(s["temperature"] > 0)
    t = torch.where(greedy, 1.0, s["temperature"])[:, None]
    k = torch.where(greedy, 1, torch.where(s["top_k"] <= 0, vocab, s["top_k"].clamp(max=vocab))).long()[:, None]
    top = x.amax(1, keepdim=True)
    e = torch.exp(-torch.where(x == top, 0.0, (top - x) / t))
    w = (e * 2.0 ** 32).long()  # masses are whole numbers: no sum depends on its order
    order = torch.sort(x, dim=1, descending=True, stable=True).indices
    ws = w.gather(1, order)
    rank = torch.arange(vocab, device=x.device)[None]
    cum = torch.where(rank < k, ws, 0).cumsum(1)
    p24 = (s["top_p"].clamp(0, 1) * 2.0 ** 24).long()[:, None]
    limit = torch.where(p24 >= 1 << 24, cum[:, -1:] + 1, _part(cum[:, -1:], p24))
    keep = (rank < k) & (cum - ws < limit) & (e.gather(1, order) >= s["min_p"][:, None])
    n = keep.sum(1).clamp(min=1)
    total = cum.gather(1, n[:, None] - 1)
    u24 = (s["uniform"].clamp(0, 1) * 2.0 ** 24).long().clamp(max=(1 << 24) - 1)[:, None]
    kept = torch.zeros_like(w).scatter_(1, order, torch.where(rank < n[:, None], ws, 0))
    ids = (kept.cumsum(1) <= _part(total, u24)).sum(1)
    ids = ids.clamp(max=vocab - 1)
    prob = w.gather(1, ids[:, None])[:, 0].float() / w.sum(1).float()
    some = top[:, 0] > -math.inf
    return (torch.where(some, ids, -1).int(), torch.where(some, prob, 0.0), torch.where(some, n, 0).int())


# -------------------------------------------------------------- in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "sample":
        return _exact_sample(s)
    new, lengths = _lengths(case)
    if case["op"] == "append":
        return _exact_quantised(s["k"], case), _exact_quantised(s["v"], case)
    p, d, kv, group = case["page"], case["dim"], case["kv_heads"], case["heads"] // case["kv_heads"]
    half, g = d // 2, d // GROUP
    kinds = DTYPES[case["type"]]
    out, at = [], 0
    for b, (n, length) in enumerate(zip(new, lengths)):
        blocks = s["pool"][s["table"][b, :-(-length // p)].long()]  # [pages, kv, block]
        heads = []
        for h in range(kv):
            flat = blocks[:, h]
            kv_values = []
            for part in (0, 1):
                byte = flat[:, part * p * half:(part + 1) * p * half].reshape(-1, half).to(torch.int64)
                o = 2 * p * half + part * p * g * 4
                pair = flat[:, o:o + p * g * 4].contiguous().view(kinds).reshape(-1, g, 2).double()
                code = torch.empty(byte.shape[0], d, dtype=torch.float64, device=byte.device)
                code[:, 0::2], code[:, 1::2] = (byte % 16).double(), (byte // 16).double()
                value = pair[:, :, 1].repeat_interleave(GROUP, 1) + pair[:, :, 0].repeat_interleave(GROUP, 1) * code
                kv_values.append(value[:length])
            k, v = kv_values
            q = s["q"][at:at + n, h * group:(h + 1) * group].double()
            pos = torch.arange(length - n, length, device=k.device)[:, None, None]
            key = torch.arange(length, device=k.device)
            dots = torch.einsum("ngd,td->ngt", q, k) / math.sqrt(d)
            hidden = key > pos
            if case["window"]:
                hidden = hidden | ((pos - key >= case["window"]) & (key >= case["sinks"]))
            heads.append(torch.softmax(dots.masked_fill(hidden, -math.inf), -1) @ v)
        out.append(torch.stack(heads, 1).flatten(1, 2))
        at += n
    return torch.cat(out)


def _exact_quantised(x, case):
    x = x.double().unflatten(-1, (-1, GROUP))
    low = x.amin(-1, keepdim=True)
    step = ((x.amax(-1, keepdim=True) - low) / 15).to(DTYPES[case["type"]]).double()
    code = torch.where(step > 0, torch.round((x - low) / torch.where(step > 0, step, 1)), 0).clamp(0, 15)
    return (low + step * code).flatten(-2)


def _exact_sample(s):
    x = s["logits"].double()
    ids, probs, counts = [], [], []
    for r in range(x.shape[0]):
        t, k = float(s["temperature"][r]), int(s["top_k"][r])
        if t <= 0:
            t, k = 1.0, 1
        prob = torch.softmax(x[r] / t, 0)
        value, order = torch.sort(x[r], descending=True, stable=True)
        inside = prob[order]
        n = min(k, len(inside)) if k > 0 else len(inside)
        before = inside[:n].cumsum(0) - inside[:n]
        p = float(s["top_p"][r])
        if p < 1:
            n = max(1, int((before < p * inside[:n].sum()).sum()))
        n = max(1, min(n, int((inside >= float(s["min_p"][r]) * inside[0]).sum())))
        mass = torch.zeros_like(prob)
        mass[order[:n]] = inside[:n]
        run_ = mass.cumsum(0)
        at = int((run_ <= float(s["uniform"][r]) * run_[-1]).sum())
        at = min(at, len(run_) - 1)
        ids.append(at)
        probs.append(prob[at])
        counts.append(n)
    dev = x.device
    return (torch.tensor(ids, device=dev, dtype=torch.int32), torch.stack(probs),
            torch.tensor(counts, device=dev, dtype=torch.int32))
