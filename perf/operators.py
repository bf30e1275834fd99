"""The operators on device memory that a server's own loop calls, as cases that can be timed: a cache in pages that is
quantised as it is written and read back, attention of new tokens over it, and sampling.

`own` says whose calls `run` makes: the framework's, or the same mathematics in elementary torch operations.
"""
import math
import os
import random
import sys

import numpy as np
import torch

own = False

# heads and kv heads of the three presets and of the parity tests' small geometry
HEADS = {"7B": (32, 32), "13B": (40, 40), "70B": (64, 8), "small": (8, 2)}
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CELL = {"i8": 1, "e4m3": 1, "f16": 2, "bf16": 2}
SMALLEST = 2.0 ** -60  # a row of smaller values is written as zeros


def _attention(name, model, cache, type, page, seqs, context, chunk, mixed=False, window=0, sinks=0, head_size=128):
    heads, kv_heads = HEADS[model]
    return {"name": name, "kind": "attention", "heads": heads, "kv_heads": kv_heads, "head_size": head_size, "cache": cache, "type": type,
            "page": page, "seqs": seqs, "context": context, "chunk": chunk, "mixed": mixed, "window": window, "sinks": sinks}


def _cache(name, kind, model, cache, type, page, seqs, context, chunk, head_size=128):
    return {"name": name, "kind": kind, "kv_heads": HEADS[model][1], "head_size": head_size, "cache": cache, "type": type, "page": page,
            "seqs": seqs, "context": context, "chunk": chunk, "mixed": False}


def _sample(name, rows, vocab, type, temperature, top_k, top_p, min_p):
    """The four as texts, "a/b": a request's value is one of them, in turn."""
    return {"name": name, "kind": "sample", "rows": rows, "vocab": vocab, "type": type, "temperature": temperature, "top_k": top_k,
            "top_p": top_p, "min_p": min_p}


def listed():
    return [
        # A decode step's new rows of 16 requests in one layer of 70B, in 8-bit integers: latency is all.
        _cache("write_step", "write", "70B", "i8", "f32", 64, 16, 2000, 1),
        # The prompts of some requests at once, 7B's heads, in e4m3, from 16-bit projections.
        _cache("write_prompts", "write", "7B", "e4m3", "f16", 32, 5, 2048, 2048),
        # One request's first page and a bit, into the fp32 that the token loop works in.
        _cache("read_prefix", "read", "70B", "i8", "f32", 64, 1, 77, 77),
        # Whole requests of 13B read back, as for moving them to another server.
        _cache("read_requests", "read", "13B", "f16", "f16", 128, 6, 3000, 3000),
        # One token behind a short context: the least attention there is, 70B's heads.
        _attention("attend_one_short", "70B", "i8", "f32", 64, 1, 500, 1),
        # A decode step of 32 requests behind ragged contexts, grouped queries, 8-bit floats.
        _attention("attend_step_batch", "70B", "e4m3", "bf16", 64, 32, 4096, 1),
        # One request behind a very long context, a kv head for each query head: bytes are all.
        _attention("attend_one_long", "7B", "i8", "f32", 128, 1, 60001, 1),
        # A chunk of a prompt behind a long context, as servers cut prompts.
        _attention("attend_chunk", "70B", "i8", "f16", 64, 1, 8000, 512),
        # A whole prompt with a window and the first four tokens, in 16 bits.
        _attention("attend_prompt_window", "7B", "bf16", "bf16", 32, 2, 4096, 4096, window=1024, sinks=4),
        # Chunks of some requests beside single tokens of others, in the fp32 that the token loop works in.
        _attention("attend_mixed", "13B", "f16", "f32", 16, 12, 2500, 200, mixed=True, window=2000, sinks=16),
        # One request's next token, as a chat samples it, from fp32 logits.
        _sample("sample_one", 1, 32000, "f32", "0.8", "0", "0.95", "0"),
        # A step of many requests with settings of their own.
        _sample("sample_batch", 256, 32000, "f32", "0.7/1/0/1.3", "40/0/0/200", "0.9/1/0.95", "0/0.05"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("write", "read", "attention", "attention", "attention", "sample"))
    if kind == "sample":
        vocab = _log(rng, 100, 150000)
        pick = lambda *of: "/".join(str(rng.choice(of)) for _ in range(rng.randint(1, 3)))  # noqa: E731
        return {"kind": kind, "rows": min(_log(rng, 1, 256), 8192000 // vocab), "vocab": vocab, "type": rng.choice(tuple(TYPES)),
                "temperature": pick("0", "0.3", "0.7", "1", "1.5"), "top_k": pick("0", "0", "1", "20", "50", "1000"),
                "top_p": pick("1", "0.5", "0.9", "0.99"), "min_p": pick("0", "0", "0.02", "0.3")}
    heads, kv_heads = HEADS[rng.choice(tuple(HEADS))]
    head_size = rng.choice((128, 128, 64))
    case = {"kind": kind, "kv_heads": kv_heads, "head_size": head_size, "cache": rng.choice(tuple(CELL)), "type": rng.choice(tuple(TYPES)),
            "page": rng.choice((16, 32, 64, 128, 256))}
    width = kv_heads * head_size
    if kind != "attention":
        seqs = _log(rng, 1, 40)
        context = _log(rng, 1, max(2, min(4096, 2 ** 25 // (width * seqs))))
        whole = kind == "read" or rng.random() < 0.5
        case.update(seqs=seqs, context=context, chunk=context if whole else min(context, rng.randint(1, 3)), mixed=False)
        return case
    case["heads"] = heads
    shape = rng.choice(("step", "chunk", "prompt"))
    if shape == "step":
        context = _log(rng, 1, 60000)
        seqs = _log(rng, 1, max(1, min(64, 2 ** 27 // (width * context))))
        chunk = rng.choice((1, 1, 1, 2, 5))
    elif shape == "chunk":
        context = _log(rng, 64, 8000)
        seqs = _log(rng, 1, max(1, min(12, 2 ** 26 // (width * context))))
        chunk = _log(rng, 6, min(512, context))
    else:
        context = chunk = _log(rng, 6, 3000)
        seqs = _log(rng, 1, max(1, min(6, 2 ** 25 // (width * context))))
    case.update(seqs=seqs, context=context, chunk=min(chunk, context), mixed=shape == "chunk" and rng.random() < 0.5,
                window=_log(rng, 1, 4000) if rng.random() < 0.4 else 0, sinks=0)
    if case["window"]:
        case["sinks"] = rng.choice((0, 1, 4, 30, 64))
    return case


# ---- what a program has in hand -------------------------------------------------------------------------------


def _lengths(case):
    """New rows and positions of each sequence: the first has the longest of both, a mixed batch has every other one at a
    single token."""
    r = random.Random("%d %d %d" % (case["seqs"], case["context"], case["chunk"]))
    new, length = [case["chunk"]], [case["context"]]
    whole = case["chunk"] == case["context"]
    for i in range(1, case["seqs"]):
        n = max(1, int(case["context"] * r.uniform(0.12, 1.0)))
        length.append(n)
        if whole:
            new.append(n)
        elif case["mixed"] and i % 2:
            new.append(1)
        else:
            new.append(max(1, min(n, int(case["chunk"] * r.uniform(0.3, 1.0) + 0.5))))
    return new, length


def _rows(case, seed):
    """Keys and values as layers produce them: a few channels of large keys, and tokens of different magnitudes."""
    new, length = _lengths(case)
    n = sum(length) if case["kind"] == "attention" else sum(new)
    g = torch.Generator(device="cuda").manual_seed(seed)
    shape = (n, case["kv_heads"], case["head_size"])
    channel = torch.exp(0.4 * torch.randn(shape[1:], generator=g, device="cuda"))
    size = torch.exp(0.3 * torch.randn((n, shape[1], 1), generator=g, device="cuda"))
    k = torch.randn(shape, generator=g, device="cuda") * channel
    v = torch.randn(shape, generator=g, device="cuda") * size
    t = TYPES[case["type"]]
    k, v = k.to(t), v.to(t)
    q = None
    if case["kind"] == "attention":
        q = torch.randn((sum(new), case["heads"], case["head_size"]), generator=g, device="cuda").to(t)
    # pages in no order, each sequence with enough for its positions
    page = case["page"]
    need = [-(-x // page) for x in length]
    order = torch.randperm(sum(need), generator=g, device="cuda", dtype=torch.int32)
    table = torch.full((len(length), max(need)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, m in enumerate(need):
        table[i, :m] = order[at:at + m]
        at += m
    return k, v, q, table, sum(need)


def _starts(counts):
    return torch.tensor([0] + list(np.cumsum(counts)), dtype=torch.int32, device="cuda")


def prepare(case, seed):
    s = {"case": case, "kind": case["kind"]}
    if case["kind"] == "sample":
        logits, u, settings = _logits(case, seed)
        s.update(logits=logits, u=u, ids=torch.empty(case["rows"], dtype=torch.int32, device="cuda"), **settings)
        return s
    new, length = _lengths(case)
    k, v, q, table, n_pages = _rows(case, seed)
    s.update(k=k, v=v, q=q, table=table, new=new, length=length, starts=_starts(new),
             lengths=torch.tensor(length, dtype=torch.int32, device="cuda"))
    if own:
        sys.path.insert(0, os.path.join(os.getcwd(), "llama2.rs_amd"))
        from llama2_rs import _lib, ops
        s["type"] = {"f32": _lib.F32, "f16": _lib.F16, "bf16": _lib.BF16}[case["type"]]
        s["pool"] = pool = ops.KvPool(1, n_pages, case["page"], case["kv_heads"], case["head_size"], case["cache"])
        s["batch"] = ops.KvBatch(s["starts"].data_ptr(), s["lengths"].data_ptr(), table.data_ptr(), len(new), table.shape[1],
                                 sum(new), max(new), max(length))
        if case["kind"] != "write":  # the cache as earlier steps have left it
            starts = _starts(length)
            whole = ops.KvBatch(starts.data_ptr(), s["lengths"].data_ptr(), table.data_ptr(), len(new), table.shape[1], sum(length),
                                max(length), max(length))
            pool.write(0, whole, k.data_ptr(), v.data_ptr(), s["type"], stream=torch.cuda.current_stream().cuda_stream)
            torch.cuda.synchronize()
        if case["kind"] == "attention":
            s["out"] = torch.empty_like(q)
            s["window"], s["sinks"] = case["window"], case["sinks"]
            need = pool.attention_workspace(s["batch"], case["heads"], s["type"], window=s["window"], sinks=s["sinks"])
            s["workspace"] = torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")
    else:
        s["pool"] = pool = _pool(case, n_pages)
        if case["kind"] != "write":
            _write(pool, _slots(table, length, length, case["page"]), k, v)
    if case["kind"] != "write":
        s["k"] = s["v"] = None
    if case["kind"] != "attention":
        rows = (sum(new), case["kv_heads"], case["head_size"])
        s["k_back"], s["v_back"] = (torch.empty(rows, dtype=TYPES[case["type"]], device="cuda") for _ in "kv")
    return s


def run(s):
    if own:
        return _run_own(s)
    case, kind = s["case"], s["kind"]
    if kind == "sample":
        return _sample_plain(s["logits"], s["u"], s["temperature"], s["top_k"], s["top_p"], s["min_p"])
    pool, table, page = s["pool"], s["table"], case["page"]
    if kind == "attention":
        return _attention_plain(pool, table, s["q"], s["new"], s["length"], case)
    slots = _slots(table, s["new"], s["length"], page)
    if kind == "write":
        _write(pool, slots, s["k"], s["v"])
    return [x.to(TYPES[case["type"]]) for x in _read(pool, slots)]


def _run_own(s):
    kind = s["kind"]
    stream = torch.cuda.current_stream().cuda_stream
    if kind == "sample":
        if "call" not in s:
            sys.path.insert(0, os.path.join(os.getcwd(), "llama2.rs_amd"))
            from llama2_rs import _lib, ops
            s["call"], s["type"] = ops.sample_device, {"f32": _lib.F32, "f16": _lib.F16, "bf16": _lib.BF16}[s["case"]["type"]]
        logits = s["logits"]
        s["call"](logits.data_ptr(), logits.shape[0], logits.shape[1], s["ids"].data_ptr(), s["u"].data_ptr(), s["temperature"].data_ptr(),
                  s["top_k"].data_ptr(), s["top_p"].data_ptr(), s["min_p"].data_ptr(), type=s["type"], stream=stream)
        return s["ids"]
    pool, batch = s["pool"], s["batch"]
    if kind == "attention":
        work = s["workspace"]
        pool.attention(0, batch, s["q"].data_ptr(), s["out"].data_ptr(), s["case"]["heads"], s["type"], window=s["window"], sinks=s["sinks"],
                       workspace=work.data_ptr(), workspace_bytes=work.shape[0], stream=stream)
        return s["out"]
    if kind == "write":
        pool.write(0, batch, s["k"].data_ptr(), s["v"].data_ptr(), s["type"], stream=stream)
    pool.read(0, batch, s["k_back"].data_ptr(), s["v_back"].data_ptr(), s["type"], stream=stream)
    return [s["k_back"], s["v_back"]]


# ---- the cache, plainly ---------------------------------------------------------------------------------------


def _pool(case, n_pages):
    """Pages of rows: what is held of each value, and the rows' scales."""
    held = {"i8": torch.int8, "e4m3": torch.float8_e4m3fn, "f16": torch.float16, "bf16": torch.bfloat16}[case["cache"]]
    rows = (n_pages * case["page"], case["kv_heads"])
    pool = {"cache": case["cache"]}
    for x in "kv":
        pool[x] = torch.zeros(rows + (case["head_size"],), dtype=torch.uint8, device="cuda").view(held) if CELL[case["cache"]] == 1 else \
            torch.zeros(rows + (case["head_size"],), dtype=held, device="cuda")
        pool[x + "_scale"] = torch.zeros(rows, device="cuda")
    return pool


def _slots(table, new, length, page):
    """Where the last new[i] positions of each sequence lie."""
    at = []
    for i, (n, end) in enumerate(zip(new, length)):
        t = torch.arange(end - n, end, device=table.device)
        at.append(table[i][t // page].long() * page + t % page)
    return torch.cat(at)


def _quantise(x, cache):
    """Codes, as the numbers that they are, and scales.  The quotients in 64 bits: a code changes at a border."""
    most = {"i8": 127.0, "e4m3": 448.0}[cache]
    x = x.float()
    a = x.abs().amax(-1, keepdim=True)
    fine = torch.isfinite(a)
    # by a tensor: by a number, torch multiplies by its reciprocal, and a scale a step off turns the ties among 16-bit values round
    scale = torch.where(fine & (a >= SMALLEST), a / torch.full_like(a, most), torch.zeros_like(a))
    y = torch.where(scale > 0, x.double() / scale.double(), torch.zeros_like(x, dtype=torch.float64))
    if cache == "e4m3":
        exponent = torch.frexp(y)[1] - 1
        step = torch.exp2((torch.clamp(exponent, min=-6) - 3).double())
        y = torch.round(y / step) * step
    else:
        y = torch.round(y)
    y = torch.clamp(y, -most, most)
    return y.float(), torch.where(fine, scale, torch.full_like(scale, math.nan)).squeeze(-1)


def _write(pool, slots, k, v):
    for name, x in (("k", k), ("v", v)):
        if pool["cache"] in ("i8", "e4m3"):
            codes, scale = _quantise(x, pool["cache"])
            held = codes.to(pool[name].dtype)
            pool[name].view(torch.uint8)[slots] = held.view(torch.uint8)
            pool[name + "_scale"][slots] = scale
        else:
            pool[name][slots] = x.float().to(pool[name].dtype)


def _read(pool, slots):
    out = []
    for name in "kv":
        if pool["cache"] in ("i8", "e4m3"):
            codes = pool[name].view(torch.uint8)[slots].view(pool[name].dtype).float()
            out.append(codes * pool[name + "_scale"][slots].unsqueeze(-1))
        else:
            out.append(pool[name][slots].float())
    return out


def _attention_plain(pool, table, q, new, length, case):
    heads, kv_heads, d = case["heads"], case["kv_heads"], case["head_size"]
    group = heads // kv_heads
    out = torch.empty_like(q)
    at = 0
    for i, (n, end) in enumerate(zip(new, length)):
        slots = _slots(table[i:i + 1], [end], [end], case["page"])
        k, v = _read(pool, slots)
        k, v = k.permute(1, 2, 0).contiguous(), v.permute(1, 0, 2).contiguous()  # [kv head][d][t] and [kv head][t][d]
        rows = q[at:at + n].float().view(n, kv_heads, group, d).permute(1, 2, 0, 3).reshape(kv_heads, group * n, d) * (1.0 / math.sqrt(d))
        pos = torch.arange(end - n, end, device=q.device).unsqueeze(1)
        t = torch.arange(end, device=q.device)
        seen = t <= pos
        if case["window"]:
            seen &= (t > pos - case["window"]) | (t < case["sinks"])
        seen = seen.repeat(group, 1)
        each = max(1, 2 ** 28 // (group * n * end))  # kv heads at a time
        for h in range(0, kv_heads, each):
            s = torch.matmul(rows[h:h + each], k[h:h + each])
            s = s.masked_fill(~seen, -math.inf)
            p = torch.exp(s - s.amax(-1, keepdim=True))
            o = torch.matmul(p / p.sum(-1, keepdim=True), v[h:h + each])
            m = o.shape[0]
            o = o.view(m, group, n, d).permute(2, 0, 1, 3).reshape(n, m * group, d)
            out[at:at + n, h * group:(h + m) * group] = o.to(q.dtype)
        at += n
    return out


# ---- sampling, plainly ----------------------------------------------------------------------------------------


def _logits(case, seed):
    """Logits as trained models have them: a wide bell, and some tokens that the context speaks for."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    rows, vocab = case["rows"], case["vocab"]
    logits = 2.0 * torch.randn((rows, vocab), generator=g, device="cuda")
    many = min(24, vocab)
    at = torch.randint(0, vocab, (rows, many), generator=g, device="cuda")
    logits.scatter_add_(1, at, 9.0 * torch.rand((rows, many), generator=g, device="cuda"))
    settings = {}
    for name, t in (("temperature", torch.float32), ("top_k", torch.int32), ("top_p", torch.float32), ("min_p", torch.float32)):
        of = [float(x) for x in case[name].split("/")]
        settings[name] = torch.tensor([of[i % len(of)] for i in range(rows)], device="cuda").to(t)
    u = torch.randint(0, 1 << 24, (rows,), generator=g, device="cuda").float() / float(1 << 24)
    return logits.to(TYPES[case["type"]]), u, settings


def _sample_plain(logits, u, temperature, top_k, top_p, min_p):
    rows, vocab = logits.shape
    x, order = torch.sort(logits.double(), dim=1, descending=True, stable=True)
    t = temperature.double().unsqueeze(1)
    w = torch.exp((x - x[:, :1]) / torch.where(t > 0, t, torch.ones_like(t)))
    place = torch.arange(vocab, device=logits.device).unsqueeze(0)
    k = top_k.unsqueeze(1)
    kept = (place < k) | (k <= 0) | (k >= vocab)
    w = torch.where(kept, w, torch.zeros_like(w))
    total = torch.cumsum(w, 1)
    p = top_p.double().unsqueeze(1)
    kept &= (total - w < p * total[:, -1:]) | (place == 0) | (p >= 1)
    kept &= (w >= min_p.double().unsqueeze(1)) | (place == 0)
    kept &= (t > 0) | (place == 0)
    # back in the vocabulary's order: the first token behind which the weights pass u of the whole
    by_id = torch.zeros_like(w).scatter_(1, order, torch.where(kept, w, torch.zeros_like(w)))
    total = torch.cumsum(by_id, 1)
    passed = total > u.double().unsqueeze(1) * total[:, -1:]
    return torch.where(passed, place, torch.full_like(place, vocab)).amin(1).int()


# ---- from the definition, in 64 bits --------------------------------------------------------------------------


def _values64(x, cache):
    """What the cache stands for once x has been written: rows over the last axis."""
    if cache in ("f16", "bf16"):
        return x.float().to(TYPES[cache]).double()
    most = 127 if cache == "i8" else 448
    x = x.double()
    scale = (x.abs().max(dim=-1).values / most).float().double().unsqueeze(-1)
    scale = torch.where(scale * most < SMALLEST * 0.999, torch.zeros_like(scale), scale)
    y = torch.nan_to_num(x / scale, 0.0)
    if cache == "i8":
        return y.round() * scale
    # e4m3: a grid of eight steps to a power of two down to 2^-6, steps of 2^-9 below
    low = torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6)))
    low = torch.where(torch.pow(2.0, low + 1) <= y.abs(), low + 1, low)
    grid = torch.pow(2.0, low - 3)
    return (y / grid).round() * grid * scale


def exact(case, seed):
    if case["kind"] == "sample":
        return _exact_ids(case, seed)
    k, v, q, _, _ = _rows(case, seed)
    k, v = _values64(k, case["cache"]), _values64(v, case["cache"])
    new, length = _lengths(case)
    if case["kind"] != "attention":
        return [k, v]
    group = case["heads"] // case["kv_heads"]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    row = at = 0
    for n, end in zip(new, length):
        for i0 in range(0, n, 1024):
            i1 = min(n, i0 + 1024)
            pos = torch.arange(end - n + i0, end - n + i1, device=q.device)[:, None]
            t = torch.arange(end, device=q.device)[None]
            hidden = t > pos
            if case["window"]:
                hidden = hidden | ((pos - t >= case["window"]) & (t >= case["sinks"]))
            for h in range(case["heads"]):
                score = q[row + i0:row + i1, h].double() @ k[at:at + end, h // group].T / case["head_size"] ** 0.5
                score[hidden] = -math.inf
                out[row + i0:row + i1, h] = torch.softmax(score, -1) @ v[at:at + end, h // group]
        row += n
        at += end
    return out


def _exact_ids(case, seed):
    logits, u, settings = _logits(case, seed)
    x, u = logits.float().cpu().numpy().astype(np.float64), u.cpu().numpy().astype(np.float64)
    settings = {name: a.cpu().numpy() for name, a in settings.items()}
    ids = np.empty(len(x), np.int32)
    for i, row in enumerate(x):
        t, k, p, least = (float(settings[name][i]) for name in ("temperature", "top_k", "top_p", "min_p"))
        order = np.argsort(-row, kind="stable")
        if t <= 0:
            ids[i] = order[0]
            continue
        if 0 < k < len(row):
            order = order[:int(k)]
        w = np.exp((row[order] - row[order[0]]) / t)
        if p < 1:
            order = order[:int(np.searchsorted(np.cumsum(w), p * w.sum())) + 1]
        w = w[:len(order)]
        order = np.sort(order[w >= min(least, 1.0)])
        cdf = np.cumsum(np.exp((row[order] - row.max()) / t))
        ids[i] = order[min(len(order) - 1, int(np.searchsorted(cdf, u[i] * cdf[-1], side="right")))]
    return torch.from_numpy(ids)


# ---- what a pass cannot do without ----------------------------------------------------------------------------


def work(case):
    size = {"f32": 4, "f16": 2, "bf16": 2}
    if case["kind"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * size[case["type"]] + 24 * case["rows"], "flops": 4 * n}
    new, length = _lengths(case)
    width = case["kv_heads"] * case["head_size"]
    scales = 4 * case["kv_heads"] if CELL[case["cache"]] == 1 else 0
    held = 2 * (width * CELL[case["cache"]] + scales)  # a position's key and value as the cache holds them
    value = 2 * width * size[case["type"]]
    if case["kind"] == "write":  # written, and read back
        return {"bytes": sum(new) * (2 * value + 2 * held), "flops": 4 * sum(new) * width}
    if case["kind"] == "read":
        return {"bytes": sum(new) * (value + held), "flops": 2 * sum(new) * width}
    window, sinks = case["window"] or 1 << 40, case["sinks"]
    pairs = positions = 0
    for n, end in zip(new, length):
        pos = np.arange(end - n, end, dtype=np.int64)
        inside = np.minimum(pos + 1, window)
        pairs += int(inside.sum() + np.minimum(sinks, pos + 1 - inside).sum())
        first = max(0, end - n - window + 1)
        positions += end - first + min(sinks, first)
    rows = 2 * sum(new) * case["heads"] * case["head_size"] * size[case["type"]]
    return {"bytes": positions * held + rows, "flops": 4 * pairs * case["heads"] * case["head_size"]}
