"""Decoding many continuations behind one prefix: the operators' measured cases.

Three operators, each through the C ABI over device pointers (include/aotk.h):

  sinks   aotk_attention_sinks: rows of one sequence over its cache, each row
          seeing a sliding window of the latest positions and the first few
          positions of all ("sinks"); single tokens and prompts;
  shared  aotk_attention_shared: rows of a batch of sequences, each behind the
          same prefix (read once for all) and a tail of its own, ragged in
          length and in rows;
  rules   aotk_logits_rules: repetition / presence / frequency penalties over a
          token history, sparse biases and a mask of allowed tokens on the
          logits of a batch, with each row's greedy pick.

`own` selects the framework's entry points; otherwise `run` computes the same
in elementary torch operations in 32 bits.
"""
import ctypes as C
import math
import os
import sys

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
KINDS = {"f32": 0, "f16": 1, "bf16": 2}  # enum aotk_kind
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
# aotk_logits_rule, one per row
RULE = np.dtype([("repetition", "<f4"), ("presence", "<f4"), ("frequency", "<f4"), ("hist_off", "<u4"),
                 ("hist_len", "<u4"), ("bias_off", "<u4"), ("bias_len", "<u4"), ("mask", "<i4")])
NO_TOKEN = -1  # the pick's bits where no token is left


# ------------------------------------------------------------------- cases
def _sinks(name, kind, heads, pos0, m, window, n_sink):
    return {"name": name, "op": "sinks", "kind": kind, "n_head": heads[0], "n_kv_head": heads[1],
            "head_dim": heads[2], "pos0": pos0, "m": m, "window": window, "n_sink": n_sink}


def _shared(name, kind, heads, n_prefix, batch, tail, rows):
    return {"name": name, "op": "shared", "kind": kind, "n_head": heads[0], "n_kv_head": heads[1],
            "head_dim": heads[2], "n_prefix": n_prefix, "batch": batch, "tail": tail, "rows": rows}


def _rules(name, kind, rows, vocab, hist, bias, masked):
    return {"name": name, "op": "rules", "kind": kind, "rows": rows, "vocab": vocab, "hist": hist, "bias": bias,
            "masked": masked}


# (query heads, kv heads, head_dim) of the configurations
_TINY, _MID, _WIDE = (32, 4, 64), (32, 8, 128), (8, 4, 256)


def listed():
    return [
        # One decode step of a local layer with the framework's f32 cache, a
        # 1024-position window and the 4 sinks that streaming decoding keeps.
        _sinks("sinks_decode_f32_at_8191", "f32", _WIDE, 8191, 1, 1024, 4),
        # One decode step far into a long document, 16-bit cache.
        _sinks("sinks_decode_bf16_at_100003", "bf16", _MID, 100003, 1, 32768, 16),
        # The last 64-row chunk of a 4096-token prompt, the f32 cache.
        _sinks("sinks_prompt_f32_64_at_4032", "f32", _MID, 4032, 64, 1024, 4),
        # A whole document read at once.
        _sinks("sinks_prompt_bf16_8192", "bf16", _MID, 0, 8192, 4096, 64),
        # Four short continuations of a system prompt on a small model.
        _shared("shared_decode_f32_4_behind_512", "f32", _TINY, 512, 4, 48, 1),
        # Sixteen users of one assistant, the f32 cache.
        _shared("shared_decode_f32_16_behind_4096", "f32", _MID, 4096, 16, 256, 1),
        # Sixty-four samples of one long document's question.
        _shared("shared_decode_bf16_64_behind_8192", "bf16", _MID, 8192, 64, 512, 1),
        # Twelve requests' own prompts read behind the prefix, ragged rows.
        _shared("shared_extend_f16_12_behind_3001", "f16", _WIDE, 3001, 12, 300, 40),
        # One chat's decode step: a short history, no grammar.
        _rules("rules_f32_1x32000", "f32", 1, 32000, 38, 0, False),
        # A few long chats: histories of thousands of tokens.
        _rules("rules_f16_7x151936", "f16", 7, 151936, 8192, 300, True),
        # A batch under grammars.
        _rules("rules_f32_64x128256", "f32", 64, 128256, 2000, 32, True),
        # A large batch with the largest vocabulary.
        _rules("rules_bf16_256x262144", "bf16", 256, 262144, 512, 8, True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the listed ranges: lengths over their logarithm, odd
    ones among them, at most the largest listed case's cost."""
    op = rng.choice(("sinks", "shared", "rules"))
    kind = rng.choice(("f32", "f16", "bf16"))
    if op == "rules":
        vocab = rng.choice((32000, 128256, 151936, 262144, _log(rng, 1000, 262144)))
        rows = _log(rng, 1, 256)
        while rows * vocab * SIZE[kind] > 256 * 262144 * 2:
            rows = rows // 2
        c = _rules("", kind, rows, vocab, rng.choice((0, _log(rng, 1, 8192))), rng.choice((0, _log(rng, 1, 300))),
                   rng.random() < 0.6)
    else:
        heads = rng.choice((_TINY, _MID, _WIDE, (rng.choice((1, 2, 3, 5)) * 4, 4, 128)))
        if op == "sinks":
            m = 1 if rng.random() < 0.4 else _log(rng, 2, 8192)
            pos0 = _log(rng, 1, 100003) if m == 1 else _log(rng, 1, 8192)
            c = _sinks("", kind, heads, pos0, m, _log(rng, 16, 32768 if m == 1 else 4096),
                       rng.choice((0, 1, 4, _log(rng, 2, 64))))
            while work(c)["flops"] > (0.06 if kind == "f32" else 1.0) * _MOST["sinks"]:
                c["m"] = c["m"] // 2
        else:
            rows = 1 if rng.random() < 0.6 else _log(rng, 2, 40)
            c = _shared("", kind, heads, _log(rng, 64, 8192), _log(rng, 1, 64), _log(rng, 1, 512), rows)
            c["tail"] = max(c["tail"], c["rows"])
            while work(c)["flops"] > _MOST["shared"]:
                c["batch"] = c["batch"] // 2
    del c["name"]
    return c


def _spread(n, most, salt):
    """n lengths over 1..most, the same for every seed: a fixed scatter whose first one is `most`."""
    return [1 + (most - 1) * ((389 * i + 97 * salt) % 1000) // 999 if i else most for i in range(n)]


def _lens(case):
    """(tail_len, rows) of every sequence of a shared case."""
    n = case["batch"]
    rows = _spread(n, case["rows"], 3)
    tail = [max(t, r) for t, r in zip(_spread(n, case["tail"], 7), rows)]
    return tail, rows


# ------------------------------------------------------------------ inputs
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) & 0x7FFFFFFFFFFFFFFF)
    return g


def prepare(case, seed):
    s = _inputs(case, seed)
    # The entry points run on the library's stream, which does not wait for
    # torch's: what they read is complete, and what they write is free, here.
    torch.cuda.synchronize()
    return s


def _inputs(case, seed):
    g = _gen(seed)
    s = dict(case)
    t = DTYPES[case["kind"]]

    def randn(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(t)

    if case["op"] == "rules":
        rows, vocab = case["rows"], case["vocab"]
        rules = np.zeros(rows, RULE)
        # logits of a trained model's size; histories that repeat their tokens
        s["logits"] = randn(rows, vocab, scale=3.0)
        hist = _spread(rows, case["hist"], 5) if case["hist"] else [0] * rows
        bias = _spread(rows, case["bias"], 9) if case["bias"] else [0] * rows
        u = torch.rand(sum(hist), generator=g, device="cuda", dtype=torch.float64)
        s["hist"] = (u ** 3 * vocab).to(torch.int32)
        s["bias_id"] = torch.randint(0, vocab, (sum(bias),), generator=g, device="cuda", dtype=torch.int32)
        s["bias"] = torch.randn(sum(bias), generator=g, device="cuda") * 4
        words = (vocab + 31) // 32
        n_mask = (rows + 1) // 2 if case["masked"] else 0
        m = torch.randint(0, 1 << 32, (3, n_mask, words), generator=g, device="cuda", dtype=torch.int64)
        m = m[0] & m[1] & m[2]  # one token of eight is allowed
        s["mask"] = torch.where(m >= 1 << 31, m - (1 << 32), m).to(torch.int32)
        rules["repetition"] = np.float32(1.1) + np.arange(rows, dtype=np.float32) % 3 * np.float32(0.1)
        rules["presence"] = np.arange(rows) % 2 * 0.5
        rules["frequency"] = np.arange(rows) % 5 * 0.05
        rules["hist_len"], rules["bias_len"] = hist, bias
        rules["hist_off"], rules["bias_off"] = np.cumsum([0] + hist[:-1]), np.cumsum([0] + bias[:-1])
        # requests of one grammar share their mask; some have none
        rules["mask"] = [-1 if i % 4 == 3 else i // 2 for i in range(rows)] if n_mask else -1
        s["rules"] = rules
        s["out"] = torch.empty_like(s["logits"])
        s["tokens"] = torch.empty(rows, dtype=torch.int32, device="cuda")
        return s
    kv, hd = case["n_kv_head"], case["head_dim"]
    if case["op"] == "sinks":
        ctx = case["pos0"] + case["m"]
        n_rows = case["m"]
        s["k"], s["v"] = randn(ctx, kv, hd), randn(ctx, kv, hd)
        s["ctx"] = ctx
    else:
        tail, rows = _lens(case)
        n_rows = sum(rows)
        s["tail_len"], s["n_rows"] = np.array(tail, np.uint32), np.array(rows, np.uint32)
        s["k_prefix"], s["v_prefix"] = randn(case["n_prefix"], kv, hd), randn(case["n_prefix"], kv, hd)
        cap = max(tail) + 5
        s["k_tail"], s["v_tail"] = randn(case["batch"], cap, kv, hd), randn(case["batch"], cap, kv, hd)
        s["cap"] = cap
    # queries somewhat larger than the keys, so that the softmax has peaks
    s["q"] = randn(n_rows, case["n_head"], hd, scale=1.5)
    s["out"] = torch.empty_like(s["q"])
    return s


# --------------------------------------------------------------------- run
def _lib():
    pkg = os.path.join(os.getcwd(), "aot-llm_amd")  # run from the repository's root
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import aotk
    aotk.init(0)
    return aotk.abi


def _run_own(s):
    abi = _lib()
    lib = abi.load()
    kind = KINDS[s["kind"]]
    if s["op"] == "sinks":
        abi.check(lib.aotk_attention_sinks(
            s["out"].data_ptr(), s["q"].data_ptr(), s["k"].data_ptr(), s["v"].data_ptr(), kind, s["n_head"],
            s["n_kv_head"], s["head_dim"], s["ctx"], 0, s["pos0"], s["m"], s["window"], s["n_sink"]))
        return s["out"]
    if s["op"] == "shared":
        abi.check(lib.aotk_attention_shared(
            s["out"].data_ptr(), s["q"].data_ptr(), s["k_prefix"].data_ptr(), s["v_prefix"].data_ptr(),
            s["k_tail"].data_ptr(), s["v_tail"].data_ptr(), kind, s["n_head"], s["n_kv_head"], s["head_dim"],
            s["n_prefix"], s["n_prefix"], s["cap"], 0, s["batch"], s["tail_len"].ctypes.data, s["n_rows"].ctypes.data))
        return s["out"]
    rows, vocab = s["logits"].shape
    abi.check(lib.aotk_logits_rules(
        s["out"].data_ptr(), s["logits"].data_ptr(), kind, rows, vocab, vocab, s["rules"].ctypes.data,
        s["hist"].data_ptr(), s["hist"].numel(), s["bias_id"].data_ptr(), s["bias"].data_ptr(), s["bias"].numel(),
        s["mask"].data_ptr(), s["mask"].shape[0], s["tokens"].data_ptr()))
    return {"logits": s["out"], "tokens": s["tokens"]}


def _attend(q, k, v, visible):
    """softmax(q k^T / sqrt(d)) v in 32 bits. q [b, kv, rows, d], k and v
    [b, kv, keys, d], visible broadcast to [b, kv, rows, keys]."""
    s = torch.matmul(q, k.transpose(-1, -2).contiguous()) * (1.0 / math.sqrt(q.shape[-1]))
    s = torch.where(visible, s, torch.full_like(s[:1, :1, :1, :1], -math.inf))
    p = torch.exp(s - s.amax(-1, keepdim=True))
    return torch.matmul(p, v) / p.sum(-1, keepdim=True)


def _run_sinks(s):
    m, nh, nkv, hd = s["m"], s["n_head"], s["n_kv_head"], s["head_dim"]
    group, pos0, window = nh // nkv, s["pos0"], s["window"]
    # the positions that any row sees: the sinks, then the first row's window on
    first = max(0, pos0 + 1 - window) if window else 0
    n_sink = min(s["n_sink"], first)
    at = torch.cat([torch.arange(n_sink, device="cuda"), torch.arange(first, pos0 + m, device="cuda")])
    k = s["k"][at].float().transpose(0, 1).contiguous()[None]
    v = s["v"][at].float().transpose(0, 1).contiguous()[None]
    q = s["q"].float().view(m, nkv, group, hd).permute(1, 0, 2, 3).reshape(1, nkv, m * group, hd)
    p = torch.arange(pos0, pos0 + m, device="cuda")[:, None]
    visible = (at <= p) & ((at < s["n_sink"]) | (at > p - window) if window else (at >= 0))
    o = _attend(q, k, v, visible.repeat_interleave(group, 0))
    o = o.view(nkv, m, group, hd).permute(1, 0, 2, 3).reshape(m, nh, hd)
    return o.to(s["q"].dtype)


def _run_shared(s):
    nh, nkv, hd = s["n_head"], s["n_kv_head"], s["head_dim"]
    group, b, n_prefix = nh // nkv, s["batch"], s["n_prefix"]
    tail = torch.from_numpy(s["tail_len"].astype(np.int64)).cuda()
    rows = torch.from_numpy(s["n_rows"].astype(np.int64)).cuda()
    most, longest = int(s["n_rows"].max()), int(s["tail_len"].max())
    total = int(s["n_rows"].sum())
    # the packed rows padded to [b, most]
    i = torch.arange(most, device="cuda")
    has = i[None, :] < rows[:, None]
    at = (torch.cumsum(rows, 0) - rows)[:, None] + torch.minimum(i[None, :], rows[:, None] - 1)
    q = s["q"].float()[at].view(b, most, nkv, group, hd).permute(0, 2, 1, 3, 4).reshape(b, nkv, most * group, hd)
    j = torch.arange(longest, device="cuda")
    sees = j[None, None, :] <= (tail - rows)[:, None, None] + i[None, :, None]
    sees = torch.cat([torch.ones(b, most, n_prefix, dtype=torch.bool, device="cuda"), sees], 2)
    sees = sees.repeat_interleave(group, 1)[:, None]
    k = torch.cat([s["k_prefix"].float()[None].expand(b, -1, -1, -1), s["k_tail"][:, :longest].float()], 1)
    v = torch.cat([s["v_prefix"].float()[None].expand(b, -1, -1, -1), s["v_tail"][:, :longest].float()], 1)
    o = _attend(q, k.transpose(1, 2).contiguous(), v.transpose(1, 2).contiguous(), sees)
    o = o.view(b, nkv, most, group, hd).permute(0, 2, 1, 3, 4).reshape(b, most, nh, hd)
    return o[has].view(total, nh, hd).to(s["q"].dtype)


def _run_rules(s):
    x = s["logits"].float()
    rows, vocab = x.shape
    r = s["rules"]
    per_row = torch.from_numpy(np.stack([r["repetition"], r["presence"], r["frequency"]])).cuda()[:, :, None]
    row_of = torch.repeat_interleave(torch.arange(rows, device="cuda"), torch.from_numpy(r["hist_len"].astype(np.int64)).cuda())
    c = torch.zeros(rows, vocab, device="cuda")
    c.index_put_((row_of, s["hist"].long()), torch.ones((), device="cuda"), accumulate=True)
    y = torch.where(x > 0, x / per_row[0], x * per_row[0])
    y = y - (per_row[1] + per_row[2] * c)
    y = torch.where(c > 0, y, x)
    if s["bias"].numel():
        # the last entry of a token counts
        row_of = torch.repeat_interleave(torch.arange(rows, device="cuda"), torch.from_numpy(r["bias_len"].astype(np.int64)).cuda())
        flat = row_of * vocab + s["bias_id"].long()
        n = flat.numel()
        last = torch.full((rows * vocab,), -1, dtype=torch.int64, device="cuda")
        last = last.scatter_reduce(0, flat, torch.arange(n, device="cuda"), "amax")
        given = torch.where(last >= 0, s["bias"][last.clamp_min(0)], torch.zeros((), device="cuda"))
        y = y + given.view(rows, vocab)
    if s["mask"].shape[0]:
        of = torch.from_numpy(r["mask"].astype(np.int64)).cuda()
        t = torch.arange(vocab, device="cuda")
        word = s["mask"][of.clamp_min(0)][:, t // 32]
        allowed = ((word >> (t % 32).to(torch.int32)) & 1).bool() | (of < 0)[:, None]
        y = torch.where(allowed, y, torch.full_like(y[:1, :1], -math.inf))
    y = y.to(s["logits"].dtype)
    top, at = torch.where(torch.isnan(y), torch.full_like(y[:1, :1], -math.inf), y).float().max(1)
    first = (y.float() == top[:, None]).to(torch.int8).argmax(1)
    tokens = torch.where(top > -math.inf, first, torch.full_like(first, NO_TOKEN))
    return {"logits": y, "tokens": tokens.to(torch.int32)}


def run(state):
    if own:
        return _run_own(state)
    return {"sinks": _run_sinks, "shared": _run_shared, "rules": _run_rules}[state["op"]](state)


# -------------------------------------------------------------------- work
def work(case):
    size = SIZE[case["kind"]]
    if case["op"] == "rules":
        n = case["rows"] * case["vocab"]
        hist = sum(_spread(case["rows"], case["hist"], 5)) if case["hist"] else 0
        bias = sum(_spread(case["rows"], case["bias"], 9)) if case["bias"] else 0
        masks = (case["rows"] + 1) // 2 * ((case["vocab"] + 31) // 32) * 4 if case["masked"] else 0
        return {"bytes": 2 * size * n + 4 * hist + 8 * bias + masks + 36 * case["rows"], "flops": 2 * n}
    nh, kv, hd = case["n_head"], case["n_kv_head"] * case["head_dim"], case["head_dim"]
    if case["op"] == "sinks":
        pos0, m, window, n_sink = case["pos0"], case["m"], case["window"], case["n_sink"]
        first = max(0, pos0 + 1 - window) if window else 0
        keys = min(n_sink, first) + pos0 + m - first
        pairs = 0
        for p in (range(pos0, pos0 + m) if m <= 4 else ()):
            lo = max(0, p + 1 - window) if window else 0
            pairs += p + 1 - lo + min(n_sink, lo)
        if m > 4:
            p = np.arange(pos0, pos0 + m, dtype=np.int64)
            lo = np.maximum(0, p + 1 - window) if window else 0 * p
            pairs = int((p + 1 - lo + np.minimum(n_sink, lo)).sum())
        rows = m
    else:
        tail, n_rows = _lens(case)
        rows = sum(n_rows)
        keys = case["n_prefix"] + sum(tail)
        pairs = rows * case["n_prefix"] + sum(r * (t - r) + r * (r + 1) // 2 for t, r in zip(tail, n_rows))
    return {"bytes": size * (2 * keys * kv + 2 * rows * nh * hd), "flops": 4 * pairs * nh * hd}


_MOST = {op: max(work(c)["flops"] for c in listed() if c["op"] == op) for op in ("sinks", "shared")}


# ------------------------------------------------------------------- exact
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rules":
        return _exact_rules(s)
    nh, nkv, hd = case["n_head"], case["n_kv_head"], case["head_dim"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")

    def one(q, k, v, hidden):  # [rows, d], [keys, d], [keys, d], [rows, keys]
        score = (q.double() @ k.double().t().contiguous()) / math.sqrt(hd)
        return torch.softmax(score.masked_fill(hidden, -math.inf), 1) @ v.double()

    if case["op"] == "sinks":
        p = case["pos0"] + torch.arange(case["m"], device="cuda")[:, None]
        j = torch.arange(s["ctx"], device="cuda")[None, :]
        hidden = j > p
        if case["window"]:
            hidden |= (j >= case["n_sink"]) & (p - j >= case["window"])
        for h in range(nh):
            g = h * nkv // nh
            out[:, h] = one(s["q"][:, h], s["k"][:, g], s["v"][:, g], hidden)
        return out
    at = 0
    for b, (n, r) in enumerate(zip(s["tail_len"].tolist(), s["n_rows"].tolist())):
        k = torch.cat([s["k_prefix"], s["k_tail"][b, :n]])
        v = torch.cat([s["v_prefix"], s["v_tail"][b, :n]])
        j = torch.arange(len(k), device="cuda")[None, :]
        hidden = j >= len(k) - r + 1 + torch.arange(r, device="cuda")[:, None]
        for g in range(nkv):
            for h in range(g * nh // nkv, (g + 1) * nh // nkv):
                out[at:at + r, h] = one(s["q"][at:at + r, h], k[:, g], v[:, g], hidden)
        at += r
    return out


def _exact_rules(s):
    y = s["logits"].double()
    rows, vocab = y.shape
    bit = torch.arange(32, device="cuda", dtype=torch.int32)
    for i, r in enumerate(s["rules"]):
        a, n = int(r["hist_off"]), int(r["hist_len"])
        seen, times = torch.unique(s["hist"][a:a + n].long(), return_counts=True)
        x = y[i, seen]
        rep = float(r["repetition"])
        x = torch.where(x > 0, x / rep, x * rep)
        y[i, seen] = x - float(r["presence"]) - float(r["frequency"]) * times.double()
        a, n = int(r["bias_off"]), int(r["bias_len"])
        if n:
            given = dict(zip(s["bias_id"][a:a + n].tolist(), s["bias"][a:a + n].tolist()))
            ids = torch.tensor(list(given), device="cuda")
            y[i, ids] += torch.tensor(list(given.values()), device="cuda", dtype=torch.float64)
        if r["mask"] >= 0:
            allowed = ((s["mask"][int(r["mask"])][:, None] >> bit) & 1).reshape(-1)[:vocab].bool()
            y[i, ~allowed] = -math.inf
    return {"logits": y, "tokens": None}
