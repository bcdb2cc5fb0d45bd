"""The cached-attention and draft-verification operators, for measurement.

Each case is one pass through an operator of ``flock_b200.kv``:

  append   new f32 keys and values rounded into a cache (f32, bf16, e4m3 or
           4-bit blocks) at a position, and the stored rows read back;
  attend   queries at positions pos .. pos + queries - 1 over a cache that
           holds every key before and including them: causal, optionally
           limited to a sliding window and a few first keys that stay visible;
  verify   drafted tokens checked against the target's distribution with given
           uniform numbers, and the token that follows them.

``run`` computes them with elementary torch operations, or, where ``own`` is
true, with the framework's kernels.  ``exact`` restates each definition in 64
bits, apart from both.

The 4-bit cache.  Blocks of 32 values along the head: d = m / -8 with m the
first value of largest magnitude, code = clamp(floor(x / d + 8.5), 0, 15), the
scale d rounded to f16; a code c stands for (c - 8) d.  Byte i of a block
holds value i in its low and value i + 16 in its high nibble.  A head's 64
bytes hold the four blocks' bytes interleaved (keys: four bytes of each block
in turn; values: two bytes of each block in turn).
"""
import math

import torch

own = False

HD = 128
DTYPES = ("f32", "bf16", "fp8", "q4")
ELEM = {"f32": 4.0, "bf16": 2.0, "fp8": 1.0, "q4": 0.5 + 2 / 32}  # bytes a cached value
SCRATCH = 8 << 20
DEV = "cuda"


# ------------------------------------------------------------------- cases
def listed():
    return [
        # one decoded token's keys and values, the layer shape of the 0.6B model
        {"name": "append_token_q4", "op": "append", "dtype": "q4", "kv_heads": 8, "tokens": 1, "pos": 319, "capacity": 2048},
        # a long prompt's keys and values in one call
        {"name": "append_prompt_q4", "op": "append", "dtype": "q4", "kv_heads": 8, "tokens": 4096, "pos": 37, "capacity": 8192},
        # single-token decode a few hundred tokens in: latency
        {"name": "decode_short_q4", "op": "attend", "dtype": "q4", "heads": 16, "kv_heads": 8, "queries": 1, "pos": 319, "capacity": 2048, "window": 0, "sinks": 0},
        # single-token decode over a long conversation
        {"name": "decode_32k_q4", "op": "attend", "dtype": "q4", "heads": 16, "kv_heads": 8, "queries": 1, "pos": 32767, "capacity": 32768, "window": 0, "sinks": 0},
        # the 8B shape's decode at the longest context
        {"name": "decode_128k_q4", "op": "attend", "dtype": "q4", "heads": 32, "kv_heads": 8, "queries": 1, "pos": 131000, "capacity": 131072, "window": 0, "sinks": 0},
        # five drafted tokens and the one before them, checked in one step
        {"name": "draft_step_q4", "op": "attend", "dtype": "q4", "heads": 16, "kv_heads": 8, "queries": 6, "pos": 8185, "capacity": 16384, "window": 0, "sinks": 0},
        # a prompt chunk behind a cached conversation
        {"name": "prompt_1k_at_7k_q4", "op": "attend", "dtype": "q4", "heads": 16, "kv_heads": 8, "queries": 1024, "pos": 7168, "capacity": 8192, "window": 0, "sinks": 0},
        # decode far into a conversation that keeps a window and its first tokens, f32 and bf16 caches
        {"name": "window_decode_f32", "op": "attend", "dtype": "f32", "heads": 16, "kv_heads": 8, "queries": 1, "pos": 20001, "capacity": 20480, "window": 4096, "sinks": 4},
        {"name": "window_decode_bf16", "op": "attend", "dtype": "bf16", "heads": 32, "kv_heads": 8, "queries": 1, "pos": 65535, "capacity": 65536, "window": 1000, "sinks": 5},
        # an odd prompt chunk under a window
        {"name": "window_prompt_fp8", "op": "attend", "dtype": "fp8", "heads": 16, "kv_heads": 8, "queries": 777, "pos": 2500, "capacity": 4096, "window": 512, "sinks": 4},
        # one conversation's four drafted tokens, the model's vocabulary
        {"name": "verify_4", "op": "verify", "seqs": 1, "drafts": 4, "vocab": 151936, "draft_probs": True, "temperature": 0.8},
        # many conversations' (or candidate chains') drafts in one call, ragged
        {"name": "verify_32x7", "op": "verify", "seqs": 32, "drafts": 7, "vocab": 151936, "draft_probs": True, "temperature": 1.0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("append", "attend", "attend", "attend", "verify"))
    if op == "append":
        tokens, pos = _log(rng, 1, 4096), rng.randrange(0, 4000)
        return {"op": op, "dtype": rng.choice(DTYPES), "kv_heads": rng.choice((1, 2, 3, 4, 8)), "tokens": tokens, "pos": pos,
                "capacity": -(-(pos + tokens + rng.randrange(64)) // 16) * 16}
    if op == "verify":
        drafts = rng.randrange(0, 9)
        return {"op": op, "seqs": _log(rng, 1, 24), "drafts": drafts, "vocab": rng.choice((_log(rng, 100, 151936), 151936, 4096)),
                "draft_probs": rng.random() < 0.7, "temperature": rng.choice((0.0, 0.5, 0.7, 1.0, 1.3))}
    dtype = rng.choice(("q4", "q4", "q4", "f32", "bf16", "fp8"))
    kv_heads = rng.choice((1, 2, 4, 8))
    heads = kv_heads * rng.choice((1, 2, 2, 3, 4, 8 if kv_heads <= 2 else 2))
    if rng.random() < 0.6:
        longest = {"f32": 16000, "bf16": 32000, "fp8": 64000, "q4": 120000}[dtype]
        queries, keys = (1 if rng.random() < 0.6 else rng.randrange(2, 17)), _log(rng, 20, longest)
    else:
        heads = min(heads, 2 * kv_heads)
        queries, keys = _log(rng, 17, 900), _log(rng, 1000, 7000)
    window = 0 if rng.random() < 0.4 else _log(rng, 1, 6000)
    sinks = rng.choice((0, 1, 4, 17, 64)) if window else 0
    return {"op": op, "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "queries": queries, "pos": keys,
            "capacity": -(-(keys + queries + rng.randrange(100)) // 16) * 16, "window": window, "sinks": sinks}


# ------------------------------------------------------------------ inputs
def _normal(gen, *shape):
    return torch.randn(*shape, device=DEV, generator=gen)


def _to_cache(x, dtype, capacity):
    """f32 rows [n][heads][128] -> a cache of `capacity` keys, as the framework lays it out."""
    n, heads, _ = x.shape
    if dtype == "q4":
        codes, scales = _q4_codes(x)
        return codes, scales
    t = {"f32": torch.float32, "bf16": torch.bfloat16, "fp8": torch.float8_e4m3fn}[dtype]
    return (x.clamp(-448, 448) if dtype == "fp8" else x).to(t), None


def _empty_cache(dtype, heads, capacity):
    if dtype == "q4":
        return torch.zeros(heads, capacity, 64, dtype=torch.uint8, device=DEV), torch.zeros(heads, capacity, 4, dtype=torch.float16, device=DEV)
    t = {"f32": torch.float32, "bf16": torch.bfloat16, "fp8": torch.float8_e4m3fn}[dtype]
    return torch.zeros(capacity, heads, HD, dtype=t, device=DEV), None


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    s = dict(case)
    if case["op"] == "verify":
        n, d, v = case["seqs"], case["drafts"], case["vocab"]
        # a target's logits (a few likely tokens over a broad tail) and a
        # draft model's, which follows it loosely
        target = _normal(gen, n, d + 1, v) * 2.5
        s["target"] = target
        s["draft"] = (target[:, :d] * 0.9 + _normal(gen, n, d, v)) if case["draft_probs"] else None
        rank = s["draft"] if case["draft_probs"] else target[:, :d]
        t = case["temperature"] or 1.0
        gumbel = -torch.log(-torch.log(torch.rand(n, d, v, device=DEV, generator=gen).clamp_(1e-9, 1 - 1e-7)))
        s["ids"] = (rank / t + gumbel).argmax(-1).to(torch.int32) if d else torch.zeros(n, 0, dtype=torch.int32, device=DEV)
        if not case["temperature"] and d:  # greedy drafts agree often
            s["ids"] = torch.where(torch.rand(n, d, device=DEV, generator=gen) < 0.7, target[:, :d].argmax(-1).to(torch.int32), s["ids"])
        s["lens"] = torch.randint(0, d + 1, (n,), device=DEV, generator=gen, dtype=torch.int32) if n > 1 else torch.full((n,), d, device=DEV, dtype=torch.int32)
        s["u"] = torch.rand(n, d + 1, device=DEV, generator=gen)
        s["tokens"] = torch.zeros(n, d + 1, dtype=torch.int32, device=DEV)
        s["accepted"] = torch.zeros(n, dtype=torch.int32, device=DEV)
        s["scratch"] = torch.zeros(SCRATCH, dtype=torch.uint8, device=DEV)
        return s
    nkv, cap = case["kv_heads"], case["capacity"]
    s["k"], s["ks"] = _empty_cache(case["dtype"], nkv, cap)
    s["v"], s["vs"] = _empty_cache(case["dtype"], nkv, cap)
    if case["op"] == "append":
        n = case["tokens"]
        # normed, rotated keys with some large channels; plain values
        s["k_new"] = _normal(gen, n, nkv, HD) * (1 + 3 * (torch.rand(HD, device=DEV, generator=gen) < 0.05))
        s["v_new"] = _normal(gen, n, nkv, HD) * 0.5
        s["k_out"], s["v_out"] = torch.empty_like(s["k_new"]), torch.empty_like(s["v_new"])
        return s
    n = case["pos"] + case["queries"]
    gain = 1 + 2 * (torch.rand(HD, device=DEV, generator=gen) < 0.05)
    for name, sc, g in (("k", "ks", gain), ("v", "vs", 0.5)):
        for h in range(nkv):  # a head at a time: a long cache's f32 rows are large
            x, d = _to_cache(_normal(gen, n, 1, HD) * g, case["dtype"], cap)
            if case["dtype"] == "q4":
                s[name][h, :n] = _interleave(x, name)[0]
                s[sc][h, :n] = d[:, 0]
            else:
                s[name][:n, h] = x[:, 0]
    s["q"] = _normal(gen, case["queries"], case["heads"], HD)
    s["out"] = torch.empty(case["queries"], case["heads"], HD, device=DEV)
    s["scratch"] = torch.zeros(SCRATCH, dtype=torch.uint8, device=DEV)
    return s


# ----------------------------------------------------- the plain form's parts
def _q4_codes(x):
    """[n][heads][128] f32 -> codes [n][heads][4][32] and f16 scales [n][heads][4]."""
    n, heads, _ = x.shape
    b = x.clamp(-524032.0, 524032.0).view(n, heads, 4, 32).double()  # next to a border in 64 bits
    top = b.abs().argmax(-1, keepdim=True)
    d = b.gather(-1, top) / -8
    inv = torch.where(d == 0, torch.zeros_like(d), 1 / d)
    codes = (b * inv + 8.5).floor().clamp(0, 15).to(torch.uint8)
    return codes, d[..., 0].float().half()


def _interleave(codes, which):
    """codes [n][heads][4][32] -> the cache's bytes [heads][n][64]."""
    n, heads = codes.shape[:2]
    byte = codes[..., :16] | (codes[..., 16:] << 4)
    parts, width = (4, 4) if which == "k" else (8, 2)
    return byte.view(n, heads, 4, parts, width).transpose(2, 3).reshape(n, heads, 64).transpose(0, 1).contiguous()


def _values(data, scales, dtype, which, at):
    """The cached rows `at` (a slice or indices) as f32 [heads][n][128]."""
    if dtype != "q4":
        return data[at].float().transpose(0, 1)
    parts, width = (4, 4) if which == "k" else (8, 2)
    b, d = data[:, at], scales[:, at]
    heads, n = b.shape[:2]
    b = b.view(heads, n, parts, 4, width).transpose(2, 3).reshape(heads, n, 4, 16)
    codes = torch.cat((b & 15, b >> 4), -1).float() - 8
    return (codes * d.float().unsqueeze(-1)).view(heads, n, HD)


def _store(s, name, sc, at):
    x = s[name + "_new"]
    if s["dtype"] == "q4":
        codes, d = _q4_codes(x)
        s[name][:, at] = _interleave(codes, name)
        s[sc][:, at] = d.transpose(0, 1)
    else:
        s[name][at] = (x.clamp(-448, 448) if s["dtype"] == "fp8" else x).to(s[name].dtype)
    return _values(s[name], s[sc], s["dtype"], name, at).transpose(0, 1)


def _run_append(s):
    at = slice(s["pos"], s["pos"] + s["tokens"])
    return [_store(s, "k", "ks", at), _store(s, "v", "vs", at)]


def _run_attend(s):
    nq, pos, nkv, heads = s["queries"], s["pos"], s["kv_heads"], s["heads"]
    n = pos + nq
    at = slice(0, n)
    key = torch.arange(n, device=DEV)
    if s["window"]:  # the keys that some query sees
        lo = max(0, pos - s["window"] + 1)
        sinks = min(s["sinks"], lo)
        at = torch.cat((key[:sinks], key[lo:]))
        key = at
    k = _values(s["k"], s["ks"], s["dtype"], "k", at)
    v = _values(s["v"], s["vs"], s["dtype"], "v", at)
    q = s["q"].view(nq, nkv, heads // nkv, HD).permute(1, 2, 0, 3).reshape(nkv, -1, HD)
    score = torch.matmul(q, k.transpose(1, 2)) * HD ** -0.5
    if nq > 1:
        at_q = torch.arange(pos, n, device=DEV).unsqueeze(1)
        seen = key <= at_q
        if s["window"]:
            seen &= (key > at_q - s["window"]) | (key < s["sinks"])
        score = score.view(nkv, -1, nq, key.numel()).masked_fill(~seen, -math.inf).view_as(score)
    p = (score - score.amax(-1, keepdim=True)).exp()
    o = torch.matmul(p, v) / p.sum(-1, keepdim=True)
    return o.view(nkv, -1, nq, HD).permute(2, 0, 1, 3).reshape(nq, heads, HD)


def _probabilities(logits, temperature):
    e = ((logits.double() - logits.double().amax(-1, keepdim=True)) / temperature).exp()
    return e / e.sum(-1, keepdim=True)


def _run_verify(s):
    n, d, lens = s["seqs"], s["drafts"], s["lens"].long()
    target, ids, u, t = s["target"], s["ids"].long(), s["u"].double(), s["temperature"]
    rows = torch.arange(n, device=DEV)
    step = torch.arange(d, device=DEV)
    if t == 0:
        ok = target[:, :d].argmax(-1) == ids
    else:
        p = _probabilities(target, t)
        p_id = p[:, :d].gather(2, ids.unsqueeze(2)).squeeze(2)
        if s["draft"] is not None:
            q = _probabilities(s["draft"], t)
            ok = u[:, :d] * q.gather(2, ids.unsqueeze(2)).squeeze(2) < p_id
        else:
            ok = u[:, :d] < p_id
    ok = ok & (step < lens.unsqueeze(1))
    acc = ok.long().cumprod(1).sum(1)
    if t == 0:
        nxt = target[rows, acc].argmax(-1)
    else:
        w = p[rows, acc]
        if d:  # refused at acc < lens: what the target has over the draft
            bad = (acc < lens).unsqueeze(1)
            r = acc.clamp(max=d - 1)
            if s["draft"] is not None:
                rest = (w - q[rows, r]).clamp(min=0)
                rest = torch.where(rest.sum(1, keepdim=True) > 0, rest, w)
            else:
                rest = w.scatter(1, ids[rows, r].unsqueeze(1), 0.0)
                rest = torch.where(rest.sum(1, keepdim=True) > 0, rest, w)
            w = torch.where(bad, rest, w)
        c = w.cumsum(1)
        nxt = (c > u[:, d:] * c[:, -1:]).int().argmax(1)
    out = torch.full((n, d + 1), -1, dtype=torch.int32, device=DEV)
    if d:
        out[:, :d] = torch.where(step < acc.unsqueeze(1), s["ids"], out[:, :d])
    out[rows, acc] = nxt.int()
    return [out, acc.int()]


# ------------------------------------------------------------ the framework's
_device = None


def _own_device():
    global _device
    if _device is None:
        from flock_b200.lib import get_device
        _device = get_device(0)
    return _device


def _own_cache(s):
    if "cache" not in s:
        from flock_b200.kv import KVCache
        s["cache"] = KVCache(_own_device(), s["dtype"], s["kv_heads"], s["capacity"], s["k"], s["v"], s["ks"], s["vs"], workspace=s.get("scratch"))
    return s["cache"]


def _own_verify(s):
    if "verifier" not in s:
        from flock_b200.kv import DraftVerifier
        s["verifier"] = DraftVerifier(_own_device(), s["vocab"], workspace=s["scratch"])
    s["verifier"].verify(s["target"], s["draft"], s["ids"], s["u"], s["tokens"], s["accepted"], lens=s["lens"], temperature=s["temperature"])
    return [s["tokens"], s["accepted"]]


def run(state):
    op = state["op"]
    if own:
        if op == "verify":
            return _own_verify(state)
        cache = _own_cache(state)
        if op == "append":
            cache.append(state["k_new"], state["v_new"], state["pos"])
            cache.read(state["pos"], state["tokens"], state["k_out"], state["v_out"])
            return [state["k_out"], state["v_out"]]
        cache.attention(state["q"], state["pos"], state["out"], window=state["window"], sinks=state["sinks"])
        return state["out"]
    return _run_append(state) if op == "append" else _run_attend(state) if op == "attend" else _run_verify(state)


# -------------------------------------------------------------------- floors
def _pairs(case):
    """(query, key) pairs that are seen, and keys that some query sees."""
    nq, pos, w = case["queries"], case["pos"], case["window"]
    if not w:
        return sum(pos + i + 1 for i in range(nq)), pos + nq
    seen = sum(min(p + 1, w) + min(case["sinks"], max(0, p - w + 1)) for p in range(pos, pos + nq))
    lo = max(0, pos - w + 1)
    return seen, pos + nq - lo + min(case["sinks"], lo)


def work(case):
    if case["op"] == "append":  # rows in, the cache's bytes out, the stored rows out
        n = case["tokens"] * case["kv_heads"] * HD * 2
        return {"bytes": n * (4 + ELEM[case["dtype"]] + 4), "flops": 0}
    if case["op"] == "attend":
        pairs, keys = _pairs(case)
        b = keys * case["kv_heads"] * HD * 2 * ELEM[case["dtype"]] + 8 * case["queries"] * case["heads"] * HD
        return {"bytes": b, "flops": 4 * HD * pairs * case["heads"]}
    drafts = case["drafts"] / 2 if case["seqs"] > 1 else case["drafts"]  # ragged: half on average
    rows = case["seqs"] * (drafts * (2 if case["draft_probs"] and case["temperature"] else 1) + 1)
    return {"bytes": rows * case["vocab"] * 4, "flops": 0}


# --------------------------------------------------------------------- exact
def exact(case, seed):
    """Each operator's definition in 64 bits, a head, a sequence or a code at a time."""
    s = prepare(case, seed)

    def row_values(data, scales, which, head, n):  # the first n cached rows of one head, by the layout's definition
        if case["dtype"] != "q4":
            return data[:n, head].to(torch.float32).double()
        out = torch.empty(n, HD, dtype=torch.float64, device=DEV)
        raw = data[head, :n].to(torch.int32)
        for block in range(4):
            d = scales[head, :n, block].double()
            for i in range(16):
                at = 16 * (i // 4) + 4 * block + i % 4 if which == "k" else 8 * (i // 2) + 2 * block + i % 2
                out[:, 32 * block + i] = ((raw[:, at] % 16) - 8).double() * d
                out[:, 32 * block + 16 + i] = ((raw[:, at] // 16) - 8).double() * d
        return out

    def stored(x):  # what the cache keeps of x, as f32 values
        dtype = case["dtype"]
        if dtype == "f32":
            return x.clone()
        if dtype != "q4":  # the nearest with so many significant bits, ties to even
            bits, low = (8, -133) if dtype == "bf16" else (4, -9)
            x = x.double().clamp(-448, 448) if dtype == "fp8" else x.double()
            unit = torch.exp2((torch.frexp(x)[1].double() - bits).clamp(min=low))
            return (torch.round(x / unit) * unit).float()
        b = x.double().reshape(*x.shape[:-1], 4, 32)
        big = torch.maximum(b.amax(-1, keepdim=True), -b.amin(-1, keepdim=True))
        first = (b.abs() == big).int().argmax(-1, keepdim=True)
        d = torch.take_along_dim(b, first, -1) / -8
        t = b * torch.where(d == 0, torch.zeros_like(d), 1 / d)
        code = sum((t + 8.5 >= c).double() for c in range(1, 16))
        return ((code - 8) * d.float().half().double()).reshape(x.shape).float()

    def verified():
        n, d, t = s["seqs"], s["drafts"], s["temperature"]
        lens, u, ids = s["lens"].tolist(), s["u"].double().tolist(), s["ids"].tolist()
        tokens = torch.full((n, d + 1), -1, dtype=torch.int32)
        accepted = torch.zeros(n, dtype=torch.int32)
        for i in range(n):
            a = 0
            while True:
                row = s["target"][i, a].double()
                dist = torch.softmax(row / t, -1) if t else None
                if a == lens[i]:
                    break
                x = ids[i][a]
                if not t:
                    if int((row == row.max()).int().argmax()) != x:
                        break
                elif s["draft"] is None:
                    if not u[i][a] < float(dist[x]):
                        kept = dist.clone()
                        kept[x] = 0
                        dist = kept if float(kept.sum()) > 0 else dist
                        break
                else:
                    qd = torch.softmax(s["draft"][i, a].double() / t, -1)
                    if not u[i][a] * float(qd[x]) < float(dist[x]):
                        kept = torch.relu(dist - qd)
                        dist = kept if float(kept.sum()) > 0 else dist
                        break
                tokens[i, a] = x
                a += 1
            if t:
                c = torch.cumsum(dist, 0)
                tokens[i, a] = int(torch.searchsorted(c, u[i][d] * c[-1:], right=True)[0])
            else:
                tokens[i, a] = int((row == row.max()).int().argmax())
            accepted[i] = a
        return [tokens, accepted]

    if case["op"] == "append":
        return [stored(s["k_new"]), stored(s["v_new"])]
    if case["op"] == "verify":
        return verified()
    nq, pos, g = case["queries"], case["pos"], case["heads"] // case["kv_heads"]
    n = pos + nq
    out = torch.empty(nq, case["heads"], HD, dtype=torch.float64, device=DEV)
    at_q = torch.arange(pos, n, device=DEV).unsqueeze(1)
    key = torch.arange(n, device=DEV).unsqueeze(0)
    hidden = key > at_q
    if case["window"]:
        hidden = hidden | ((key <= at_q - case["window"]) & (key >= case["sinks"]))
    for kv in range(case["kv_heads"]):
        k = row_values(s["k"], s["ks"], "k", kv, n)
        v = row_values(s["v"], s["vs"], "v", kv, n)
        for h in range(kv * g, (kv + 1) * g):
            z = (s["q"][:, h].double() @ k.T) / math.sqrt(HD)
            out[:, h] = torch.softmax(torch.where(hidden, torch.full_like(z, -math.inf), z), -1) @ v
    return out
