"""The operators a token model's training step and its generation loop add to the library, as cases to measure:

  embedding   rows of a table picked by token, scaled; its gradient, added up per token
  dropout     a mask from a counter-based generator that is formed again where it is needed, with the residual sum
  attention   causal, over sequences packed one after the other, query heads in groups that share a key/value head;
              forward, forward + backward, and the few newest tokens of each sequence against its cache

``run`` computes them from elementary torch operations or, with ``own`` set, calls the library's entry points on the
same memory.  Element types are the library's two: float32 and float64.
"""
import math
import random

import numpy as np
import torch

own = False

DEVICE = "cuda"


# ---- cases ----------------------------------------------------------------------------------------------------------
def listed():
    return [
        # a first layer's lookup for a window of 49 tokens, trained in double: all latency
        {"name": "embed_train_window", "op": "embedding", "direction": "train", "type": "f64", "vocab": 1000, "width": 96, "tokens": 49},
        # a batch of sequences looked up in a large table
        {"name": "embed_lookup_batch", "op": "embedding", "direction": "forward", "type": "f32", "vocab": 50000, "width": 1024, "tokens": 16384},
        # the same layer trained: the frequent tokens have thousands of rows to add, most of the table none
        {"name": "embed_train_batch", "op": "embedding", "direction": "train", "type": "f32", "vocab": 32768, "width": 512, "tokens": 32768},
        # the activations of one window, in double
        {"name": "dropout_train_window", "op": "dropout", "direction": "train", "type": "f64", "rows": 49, "cols": 96, "p": 0.1, "residual": True},
        # a block's output joined to its input over a large batch
        {"name": "dropout_residual_batch", "op": "dropout", "direction": "forward", "type": "f32", "rows": 8192, "cols": 2048, "p": 0.1, "residual": True},
        # a few short texts, one of them a single token
        {"name": "attn_prompt_short", "op": "attention", "direction": "forward", "type": "f32", "lengths": "49,1,17,33", "heads": 3, "kv_heads": 3, "head_dim": 32},
        # a ragged batch of prompts
        {"name": "attn_prompt_packed", "op": "attention", "direction": "forward", "type": "f32", "lengths": "1024,77,513,1300,256,900,1,640,333,2048,129,700",
         "heads": 16, "kv_heads": 4, "head_dim": 64},
        # one long prompt
        {"name": "attn_prompt_long", "op": "attention", "direction": "forward", "type": "f32", "lengths": "8192", "heads": 16, "kv_heads": 4, "head_dim": 64},
        # a training batch, sequences of different lengths
        {"name": "attn_train_packed", "op": "attention", "direction": "train", "type": "f32", "lengths": "2048,1000,1536,511,300,1901,64,800",
         "heads": 16, "kv_heads": 4, "head_dim": 64},
        # a training batch in double
        {"name": "attn_train_double", "op": "attention", "direction": "train", "type": "f64", "lengths": "256,200,37,512", "heads": 6, "kv_heads": 3, "head_dim": 32},
        # one text being continued token by token: the least a step can take
        {"name": "attn_token_one", "op": "attention", "direction": "token", "type": "f32", "new": "1", "lengths": "300", "capacity": 512,
         "heads": 8, "kv_heads": 2, "head_dim": 64},
        # many texts of very different lengths being continued, one of them still empty
        {"name": "attn_token_batch", "op": "attention", "direction": "token", "type": "f32", "new": ",".join(["1"] * 24),
         "lengths": "8192,17,4096,7000,1,3000,512,6001,0,2048,8000,999,5000,64,1500,7777,2500,300,4500,8192,1200,6500,100,3500", "capacity": 8192,
         "heads": 16, "kv_heads": 4, "head_dim": 128},
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["embedding", "dropout", "attention", "attention", "attention"])
    kind = rng.choice(["f32", "f32", "f64"])
    if op == "embedding":
        width, tokens = _log_int(rng, 16, 1024), _log_int(rng, 1, 32768)
        if kind == "f64":
            width = min(width, 512)
        return {"op": op, "direction": rng.choice(["forward", "train"]), "type": kind, "vocab": _log_int(rng, 10, 32768), "width": width, "tokens": tokens}
    if op == "dropout":
        rows, cols = _log_int(rng, 1, 8192), _log_int(rng, 1, 2048 if kind == "f32" else 1024)
        return {"op": op, "direction": rng.choice(["forward", "train"]), "type": kind, "rows": rows, "cols": cols,
                "p": rng.choice([0.0, 0.05, 0.1, 0.2, 0.5]), "residual": rng.random() < 0.5}
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 4] if kv_heads < 8 else [1, 2])
    head_dim = rng.choice([16, 32, 40, 64, 64, 80, 96, 128, 128])
    direction = rng.choice(["forward", "train", "token"])
    if direction == "token":
        capacity = _log_int(rng, 16, 8192 if kind == "f32" else 2048)
        count = max(1, min(_log_int(rng, 1, 32), int(24 * 8192 * 512 / (capacity * kv_heads * head_dim) * (1.0 if kind == "f32" else 0.25))))
        most_new = rng.choice([1, 1, 1, 8, 64])
        lengths = [rng.choice([capacity, _log_int(rng, 1, capacity), rng.randint(0, capacity)]) for _ in range(count)]
        new = [min(max(1, n), rng.randint(1, most_new)) for n in lengths]
        return {"op": op, "direction": direction, "type": kind, "new": ",".join(map(str, new)), "lengths": ",".join(map(str, lengths)),
                "capacity": capacity, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim}
    room = 2.0 ** 36 / (heads * head_dim) / (3.5 if direction == "train" else 1.0) / (1.0 if kind == "f32" else 16.0)  # sequences * longest ** 2
    longest = _log_int(rng, 1, min(8192 if kind == "f32" else 1024, int(room ** 0.5)))
    count = max(1, min(_log_int(rng, 1, 24), int(room / longest ** 2)))
    lengths = [longest] + [rng.choice([_log_int(rng, 1, longest), rng.randint(0, longest)]) for _ in range(count - 1)]
    rng.shuffle(lengths)
    return {"op": op, "direction": direction, "type": kind, "lengths": ",".join(map(str, lengths)), "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim}


def _ints(text):
    return [int(x) for x in text.split(",")]


def _type(case):
    return torch.float64 if case["type"] == "f64" else torch.float32


def _starts(lengths):
    at = [0]
    for n in lengths:
        at.append(at[-1] + n)
    return at


def _pairs(new, lengths):
    """Query/key pairs that are not masked: query i of n looks at the first lengths - n + i + 1 keys."""
    return sum(sum(max(0, k - n + i + 1) for i in range(n)) for n, k in zip(new, lengths))


def work(case):
    size = 8 if case["type"] == "f64" else 4
    train = case["direction"] == "train"
    if case["op"] == "embedding":
        moved = case["tokens"] * case["width"] * size
        table = min(case["tokens"], case["vocab"]) * case["width"] * size
        return {"bytes": 4 * case["tokens"] + moved + table + (moved + case["vocab"] * case["width"] * size if train else 0),
                "flops": case["tokens"] * case["width"] * (3 if train else 1)}
    if case["op"] == "dropout":
        n = case["rows"] * case["cols"]
        return {"bytes": n * size * (2 + int(case["residual"]) + (2 if train else 0)), "flops": n * (1 + int(case["residual"]) + int(train))}
    lengths = _ints(case["lengths"])
    new = _ints(case["new"]) if case["direction"] == "token" else lengths
    q, kv = sum(new) * case["heads"] * case["head_dim"], sum(lengths) * case["kv_heads"] * case["head_dim"]
    products = 2 + (5 if train else 0)
    return {"bytes": size * (2 * q + 2 * kv + ((2 * q + 2 * kv) if train else 0)),
            "flops": 2 * products * case["head_dim"] * case["heads"] * _pairs(new, lengths)}


# ---- inputs ---------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    kind = _type(case)
    normal = lambda *shape: torch.randn(*shape, generator=g, device=DEVICE, dtype=kind)
    s = {"case": case}
    if case["op"] == "embedding":
        # tokens in the proportions of a text (the r-th most frequent about 1/r of the first), a few places without one
        u = torch.rand(case["tokens"], generator=g, device=DEVICE, dtype=torch.float64)
        rank = (torch.exp(u * math.log(case["vocab"] + 1)) - 1).long().clamp_(0, case["vocab"] - 1)
        ids = torch.randperm(case["vocab"], generator=g, device=DEVICE)[rank]
        ids[torch.rand(case["tokens"], generator=g, device=DEVICE) < 1 / 64] = -1
        s["ids"] = ids.int()
        s["table"] = normal(case["vocab"], case["width"]) * 0.02
        s["scale"] = math.sqrt(case["width"])
        s["out"] = torch.empty(case["tokens"], case["width"], device=DEVICE, dtype=kind)
        if case["direction"] == "train":
            s["d_out"], s["d_table"] = normal(case["tokens"], case["width"]), torch.empty_like(s["table"])
    elif case["op"] == "dropout":
        s["x"] = normal(case["rows"], case["cols"])
        s["residual"] = normal(case["rows"], case["cols"]) if case["residual"] else None
        s["y"] = torch.empty_like(s["x"])
        if case["direction"] == "train":
            s["dy"], s["dx"] = normal(case["rows"], case["cols"]), torch.empty_like(s["x"])
        s["seed"], s["site"] = 0x1234567 * (seed + 1), seed % 7
        s["step"] = torch.tensor([seed % 1000], device=DEVICE, dtype=torch.int32)
    else:
        heads, kv_heads, d = case["heads"], case["kv_heads"], case["head_dim"]
        lengths = _ints(case["lengths"])
        s["scale"] = 1.0 / math.sqrt(d)
        vector = lambda values: torch.tensor(values, device=DEVICE, dtype=torch.int32)
        if case["direction"] == "token":
            new = _ints(case["new"])
            s["q"] = normal(sum(new), heads * d)
            s["k"], s["v"] = normal(len(lengths) * case["capacity"], kv_heads * d), normal(len(lengths) * case["capacity"], kv_heads * d)
            begins = [i * case["capacity"] for i in range(len(lengths))]
            s["offsets"], s["k_begin"] = vector(_starts(new)), vector(begins)
            s["k_end"] = vector([b + n for b, n in zip(begins, lengths)])
            s["o"] = torch.empty_like(s["q"])
        else:
            tokens = sum(lengths)
            s["qkv"] = normal(tokens, (heads + 2 * kv_heads) * d)  # one layer's output: columns [Q | K | V]
            s["offsets"] = vector(_starts(lengths))
            s["o"] = torch.empty(tokens, heads * d, device=DEVICE, dtype=kind)
            s["lse"] = torch.empty(heads, tokens, device=DEVICE, dtype=kind)
            if case["direction"] == "train":
                s["d_o"], s["d_qkv"] = normal(tokens, heads * d), torch.empty_like(s["qkv"])
    if own:
        s["handles"] = _handles(s)
    return s


def _handles(s):
    """The library's handles on the tensors of a state, as a program that keeps its buffers makes them once."""
    from parallelreverseautodiff_amd.cudablas import CudaBlas
    from parallelreverseautodiff_amd.matrix import DeviceBuffer, IndexVector

    if not CudaBlas.Instance.IsInitialized:
        CudaBlas.Instance.Initialize()
    made = {}
    for name, t in s.items():
        if isinstance(t, torch.Tensor):
            if t.dtype == torch.int32:
                made[name] = IndexVector.wrap(t.data_ptr(), t.numel(), parent=t)
            else:
                made[name] = DeviceBuffer.wrap(np.float64 if t.dtype == torch.float64 else np.float32, t.shape[0], t.shape[1], t.data_ptr(), parent=t)
    return made


# ---- one pass -------------------------------------------------------------------------------------------------------
def run(s):
    if own:
        return _run_own(s)
    return {"embedding": _embedding, "dropout": _dropout, "attention": _attention}[s["case"]["op"]](s)


def _run_own(s):
    from parallelreverseautodiff_amd import _lib
    from parallelreverseautodiff_amd.exceptions import check

    lib, case, h = _lib.load(), s["case"], {name: b.handle for name, b in s["handles"].items()}
    train = case["direction"] == "train"
    if case["op"] == "embedding":
        check(lib.prad_embedding_fwd(h["table"], h["ids"], s["scale"], h["out"]))
        if train:
            check(lib.prad_embedding_bwd(h["d_out"], h["ids"], s["scale"], h["d_table"], 0))
        return [s["out"], s["d_table"]] if train else [s["out"]]
    if case["op"] == "dropout":
        check(lib.prad_dropout_fwd(h["x"], h.get("residual"), h["y"], case["p"], s["seed"], s["site"], h["step"]))
        if train:
            check(lib.prad_dropout_bwd(h["dy"], h["dx"], case["p"], s["seed"], s["site"], h["step"]))
        return [s["y"], s["dx"]] if train else [s["y"]]
    heads, kv_heads, d = case["heads"], case["kv_heads"], case["head_dim"]
    if case["direction"] == "token":
        check(lib.prad_cached_attention(h["q"], 0, h["k"], 0, h["v"], 0, h["o"], h["offsets"], h["k_begin"], h["k_end"], heads, kv_heads, d, s["scale"]))
        return [s["o"]]
    k_col, v_col = heads * d, (heads + kv_heads) * d
    check(lib.prad_causal_attention_fwd(h["qkv"], 0, h["qkv"], k_col, h["qkv"], v_col, h["o"], h["lse"] if train else None, h["offsets"],
                                        heads, kv_heads, d, s["scale"]))
    if not train:
        return [s["o"]]
    check(lib.prad_causal_attention_bwd(h["qkv"], 0, h["qkv"], k_col, h["qkv"], v_col, h["o"], h["lse"], h["d_o"], h["d_qkv"], 0, h["d_qkv"], k_col,
                                        h["d_qkv"], v_col, h["offsets"], heads, kv_heads, d, s["scale"]))
    return [s["o"], s["d_qkv"]]


def _embedding(s):
    ids, present = s["ids"].long().clamp(min=0), (s["ids"] >= 0)[:, None]
    out = torch.where(present, s["table"][ids] * s["scale"], 0.0)
    if s["case"]["direction"] != "train":
        return [out]
    rows = torch.where(present, s["d_out"].double(), 0.0)  # sums of thousands of rows: in double
    total = torch.zeros(s["table"].shape, device=DEVICE, dtype=torch.float64).index_add_(0, ids, rows)
    return [out, (total * s["scale"]).to(out.dtype)]


def _mask(n, p, seed, site, step):
    """Ten rounds of the counter-based generator Philox4x32 on the counters (element / 4 in two words, step, site): which
    of n elements are kept.  32-bit words in 64-bit integers; the high word of a product that wraps is still right."""
    low = 0xFFFFFFFF
    block = torch.arange((n + 3) // 4, device=DEVICE)
    c = [block & low, block >> 32, torch.zeros_like(block) + (step.long() & low), torch.full_like(block, site & low)]
    k0, k1 = seed & low, (seed >> 32) & low
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [((b >> 32) & low) ^ c[1] ^ k0, b & low, ((a >> 32) & low) ^ c[3] ^ k1, a & low]
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return torch.stack(c, dim=1).reshape(-1)[:n] >= int(math.floor(p * 4294967296.0))


def _dropout(s):
    case, x = s["case"], s["x"]
    keep = _mask(x.numel(), case["p"], s["seed"], s["site"], s["step"]).reshape(x.shape)
    factor = 1.0 / (1.0 - case["p"])
    y = torch.where(keep, x * factor, 0.0)
    if s["residual"] is not None:
        y = y + s["residual"]
    return [y, torch.where(keep, s["dy"] * factor, 0.0)] if case["direction"] == "train" else [y]


def _padded(rows, begin, count, longest):
    """[sequences, longest, ...] out of packed rows, and which of them are real."""
    at = torch.arange(longest, device=DEVICE)
    real = at[None] < count[:, None]
    return rows[torch.where(real, begin[:, None] + at[None], 0)], real


def _weights(q, k, real_k, n_q, n_k, scale):
    """softmax(q k^T scale) of padded sequences [s, kv_heads, group, i, d] and [s, kv_heads, j, d]; query i of n_q sees the
    keys up to n_k - n_q + i, a query without keys has zeros."""
    sequences, kv_heads, group, rows, d = q.shape
    scores = torch.matmul(q.reshape(sequences, kv_heads, group * rows, d), k.transpose(2, 3).contiguous()).reshape(sequences, kv_heads, group, rows, -1)
    scores *= scale
    last = torch.arange(rows, device=DEVICE)[None] + (n_k - n_q)[:, None]
    seen = (torch.arange(k.shape[2], device=DEVICE)[None, None] <= last[:, :, None]) & real_k[:, None]
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(dim=-1, keepdim=True)
    scores -= torch.where(torch.isfinite(top), top, 0.0)
    scores.exp_()
    total = scores.sum(dim=-1, keepdim=True)
    scores /= torch.where(total > 0, total, 1.0)
    return scores


def _attention(s):
    case = s["case"]
    heads, kv_heads, d = case["heads"], case["kv_heads"], case["head_dim"]
    group = heads // kv_heads
    offsets = s["offsets"].long()
    q_begin, n_q = offsets[:-1], offsets[1:] - offsets[:-1]
    lengths = _ints(case["lengths"])
    token = case["direction"] == "token"
    if token:
        q, k, v = s["q"], s["k"], s["v"]
        k_begin, n_k = s["k_begin"].long(), (s["k_end"] - s["k_begin"]).long()
    else:
        q, k, v = s["qkv"].split([heads * d, kv_heads * d, kv_heads * d], dim=1)
        k_begin, n_k = q_begin, n_q
    longest_q, longest_k = max(_ints(case["new"]) if token else lengths), max(lengths + [1])
    spread = lambda x: x.reshape(x.shape[0], x.shape[1], kv_heads, group, d).permute(0, 2, 3, 1, 4).contiguous()
    qp, real_q = _padded(q, q_begin, n_q, longest_q)
    kp, real_k = _padded(k, k_begin, n_k, longest_k)
    vp, _ = _padded(v, k_begin, n_k, longest_k)
    heads_first = lambda x: x.reshape(x.shape[0], x.shape[1], kv_heads, d).permute(0, 2, 1, 3).contiguous()
    qp, kp, vp = spread(qp), heads_first(kp), heads_first(vp)
    p = _weights(qp, kp, real_k, n_q, n_k, s["scale"])
    rows = lambda x: x.reshape(x.shape[0], kv_heads, group * longest_q, x.shape[-1])
    o = torch.matmul(rows(p), vp).reshape(qp.shape)
    packed = lambda x: x.permute(0, 3, 1, 2, 4).reshape(x.shape[0], longest_q, heads * d)[real_q]
    if case["direction"] != "train":
        return [packed(o)]
    g, _ = _padded(s["d_o"], q_begin, n_q, longest_q)
    g = spread(torch.where(real_q[:, :, None], g, 0.0))
    d_v = torch.matmul(rows(p).transpose(2, 3).contiguous(), rows(g))
    d_p = torch.matmul(rows(g), vp.transpose(2, 3).contiguous()).reshape(p.shape)
    d_p -= (g * o).sum(dim=-1, keepdim=True)
    d_s = d_p.mul_(p).mul_(s["scale"])
    d_q = torch.matmul(rows(d_s), kp).reshape(qp.shape)
    d_k = torch.matmul(rows(d_s).transpose(2, 3).contiguous(), rows(qp))
    keys = lambda x: x.permute(0, 2, 1, 3).reshape(x.shape[0], longest_k, kv_heads * d)[real_k]
    return [packed(o), torch.cat([packed(d_q), keys(d_k), keys(d_v)], dim=1)]


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {"embedding": _exact_embedding, "dropout": _exact_dropout, "attention": _exact_attention}[case["op"]](s)


def _exact_embedding(s):
    ids = s["ids"].cpu().numpy()
    table = s["table"].double().cpu().numpy()
    out = np.zeros((len(ids), table.shape[1]))
    out[ids >= 0] = table[ids[ids >= 0]] * s["scale"]
    if s["case"]["direction"] != "train":
        return [out]
    order = np.argsort(ids, kind="stable")
    order = order[ids[order] >= 0]
    d_table = np.zeros_like(table)
    if len(order):
        names, first = np.unique(ids[order], return_index=True)
        d_table[names] = np.add.reduceat(s["d_out"].double().cpu().numpy()[order], first, axis=0) * s["scale"]
    return [out, d_table]


def _exact_dropout(s):
    case, n = s["case"], s["x"].numel()
    words = np.uint64(32), np.uint64(0xFFFFFFFF)
    block = np.arange((n + 3) // 4, dtype=np.uint64)
    x0, x1 = block & words[1], block >> words[0]
    x2, x3 = np.full_like(block, int(s["step"].item()) & 0xFFFFFFFF), np.full_like(block, s["site"] & 0xFFFFFFFF)
    for r in range(10):
        key0, key1 = ((s["seed"] & 0xFFFFFFFF) + r * 0x9E3779B9) % 2 ** 32, (((s["seed"] >> 32) & 0xFFFFFFFF) + r * 0xBB67AE85) % 2 ** 32
        m0, m1 = x0 * np.uint64(0xD2511F53), x2 * np.uint64(0xCD9E8D57)
        x0, x1, x2, x3 = (m1 >> words[0]) ^ x1 ^ np.uint64(key0), m1 & words[1], (m0 >> words[0]) ^ x3 ^ np.uint64(key1), m0 & words[1]
    kept = (np.stack([x0, x1, x2, x3], axis=1).reshape(-1)[:n].astype(np.float64) >= math.floor(case["p"] * 2.0 ** 32)).reshape(s["x"].shape)
    host = lambda t: t.double().cpu().numpy()
    y = np.where(kept, host(s["x"]) / (1 - case["p"]), 0)
    if s["residual"] is not None:
        y = y + host(s["residual"])
    return [y, np.where(kept, host(s["dy"]) / (1 - case["p"]), 0)] if case["direction"] == "train" else [y]


def _exact_attention(s):
    case = s["case"]
    heads, kv_heads, d = case["heads"], case["kv_heads"], case["head_dim"]
    train, token = case["direction"] == "train", case["direction"] == "token"
    lengths = _ints(case["lengths"])
    new = _ints(case["new"]) if token else lengths
    o = torch.zeros(sum(new), heads * d, device=DEVICE, dtype=torch.float64)
    d_qkv = torch.zeros(s["qkv"].shape, device=DEVICE, dtype=torch.float64) if train else None
    for i, (at, n, m) in enumerate(zip(_starts(new), new, lengths)):
        if n == 0 or m == 0:
            continue
        keys = slice(i * case["capacity"], i * case["capacity"] + m) if token else slice(at, at + n)
        hidden = torch.ones(n, m, device=DEVICE, dtype=torch.bool).triu(m - n + 1)
        for h in range(heads):
            at_q, at_k = h * d, (h * kv_heads // heads) * d
            at_kk, at_vv = (at_k, at_k) if token else (heads * d + at_k, (heads + kv_heads) * d + at_k)
            q = (s["q"] if token else s["qkv"])[at:at + n, at_q:at_q + d].double()
            k = (s["k"] if token else s["qkv"])[keys, at_kk:at_kk + d].double()
            v = (s["v"] if token else s["qkv"])[keys, at_vv:at_vv + d].double()
            p = torch.where(hidden, -math.inf, (q @ k.T) * s["scale"])
            p = torch.where(hidden, 0.0, torch.exp(p - torch.logsumexp(p, dim=1, keepdim=True)))
            o[at:at + n, at_q:at_q + d] = p @ v
            if train:
                g = s["d_o"][at:at + n, at_q:at_q + d].double()
                pg = p * (g @ v.T)
                ds = (pg - p * pg.sum(dim=1, keepdim=True)) * s["scale"]
                d_qkv[at:at + n, at_q:at_q + d] = ds @ k
                d_qkv[keys, at_kk:at_kk + d] += ds.T @ q
                d_qkv[keys, at_vv:at_vv + d] += p.T @ g
    return [o, d_qkv] if train else [o]


if __name__ == "__main__":
    for made in listed() + [draw(random.Random(i)) for i in range(6)]:
        print(made, work(made))
