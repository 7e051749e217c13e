"""More operators of the paged cache as measurable cases: plain torch forms beside the library's calls.

* ``chunk``   ``xq_fa_chunk``: attention of a chunk of new tokens (one, a prompt, many prompts) over the
              paged cache, with a window, documents, a two-way prefix, capped scores, a bias by distance;
* ``weights`` ``xq_kv_weights``: the attention weight that each cached row has got, accumulated;
* ``evict``   ``xq_kv_pages_evict``: the rows of least weight leave the cache, in every layer's pools,
              and pages without rows are given back;
* ``verify``  ``xq_verify_tokens``: drafted tokens against the target's logits, from given random numbers.

Head shapes are the repository's own (24 query heads over 4 KV heads at head dim 256, 16 over 8 and 32
over 8 at 128), vocabularies generic. A case's lengths follow from the case alone; its values come from
the seed. Where ``own`` is false, ``run`` computes the operator from elementary torch operations in 32
bits (probabilities and their sums in 64: a drawn token lies between two of them).
"""
import ctypes
import math
import pathlib
import random
import sys

import torch

own = False

_TYPES = {"f32": 0, "f16": 1, "q4_0": 2, "q8_0": 8, "bf16": 30, "e5m2": 0x100}
_ELEM = {"f32": 4, "f16": 2, "q4_0": 18, "q8_0": 34, "bf16": 2, "e5m2": 1}
_TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "e5m2": torch.float8_e5m2}
_HEADS = {"24/4/256": (24, 4, 256), "16/8/128": (16, 8, 128), "32/8/128": (32, 8, 128)}


def _record(kv, d):
    return d // 32 * _ELEM[kv] if kv in ("q4_0", "q8_0") else d * _ELEM[kv]


def _cdiv(a, b):
    return -(-a // b)


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------

def _named(name, c):
    return {"name": name, **c} if name else c


def _chunk(name, heads, kv, kind, tokens, rows, seqs, page, ragged=False, window=0, docs=0, prefix=0, cap=0.0, bias=0.0):
    return _named(name, {"op": "chunk", "heads": heads, "kv": kv, "type": kind, "tokens": tokens, "rows": rows, "seqs": seqs,
                         "page": page, "ragged": ragged, "window": window, "docs": docs, "prefix": prefix, "cap": cap, "bias": bias})


def _weights(name, heads, kv, kind, tokens, rows, seqs, page, ragged=False, decay=1.0, window=0, cap=0.0):
    return _named(name, {"op": "weights", "heads": heads, "kv": kv, "type": kind, "tokens": tokens, "rows": rows, "seqs": seqs,
                         "page": page, "ragged": ragged, "decay": decay, "window": window, "docs": 0, "prefix": 0, "cap": cap, "bias": 0.0})


def _evict(name, heads, kv, layers, page, rows, keep, seqs, first, last, moved=False):
    return _named(name, {"op": "evict", "heads": heads, "kv": kv, "layers": layers, "page": page, "rows": rows, "keep": keep,
                         "seqs": seqs, "first": first, "last": last, "moved": moved})


def _verify(name, kind, vocab, tokens, seqs, mode, chain=False, ragged=False):
    return _named(name, {"op": "verify", "type": kind, "vocab": vocab, "tokens": tokens, "seqs": seqs, "mode": mode,
                         "chain": chain, "ragged": ragged})


def listed():
    return [
        # the last few tokens of a user's prompt on what is cached of it: latency
        _chunk("chunk_tail17_q8_f32", "24/4/256", "q8_0", "f32", 17, 500, 1, 16),
        # a decode step of 16 chats of all lengths, scores capped: one token each, fp8 cache
        _chunk("chunk_decode_cap_e5m2_b16", "16/8/128", "e5m2", "bf16", 1, 6001, 16, 64, ragged=True, cap=30.0),
        # a long prompt read in chunks: 512 more tokens on 4096 rows
        _chunk("chunk_512_f16_4k", "32/8/128", "f16", "bf16", 512, 4096, 1, 16),
        # eight users' prompts of up to 777 tokens, a sliding window, packed documents, 4-bit cache
        _chunk("chunk_window_q4_b8", "24/4/256", "q4_0", "bf16", 777, 3001, 8, 32, ragged=True, window=1024, docs=3),
        # the largest: two whole prompts of 8191 tokens
        _chunk("chunk_prompt_f16_8k_b2", "32/8/128", "f16", "bf16", 8191, 0, 2, 64),
        # a decode step's weights: 16 chats of all lengths, one f32 token each
        _weights("weights_decode_q8_b16", "24/4/256", "q8_0", "f32", 1, 8000, 16, 16, ragged=True, decay=0.99),
        # after a prompt: what its last 32 tokens look at in 16k rows, two users
        _weights("weights_last32_f16_16k_b2", "32/8/128", "f16", "bf16", 32, 16001, 2, 64),
        # every step of 32 chats at their budget: one row each makes room
        _evict("evict_step_q8_b32", "24/4/256", "q8_0", 16, 64, 2049, 2048, 32, 4, 64, moved=True),
        # after a prompt: four users' 12001 rows cut to 4096
        _evict("evict_prompt_f16_b4", "16/8/128", "f16", 8, 16, 12001, 4096, 4, 4, 32),
        # one user's chain of five drafted tokens with the draft's probabilities: latency
        _verify("verify_chain_draft_f32", "f32", 50001, 6, 1, "draft", chain=True),
        # eight users' greedy trees of up to 25 tokens
        _verify("verify_greedy_tree25_b8", "bf16", 131072, 25, 8, "greedy", ragged=True),
        # sixteen users' trees of 16 tokens, sampled
        _verify("verify_tree16_f32_b16", "f32", 128000, 16, 16, "target"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    op = rng.choice(["chunk", "chunk", "chunk", "weights", "weights", "evict", "evict", "verify", "verify"])
    heads = rng.choice(sorted(_HEADS))
    page = rng.choice([16, 16, 32, 64, 128])
    kv = rng.choice(["f16", "q8_0", "q4_0", "e5m2"])
    kind = rng.choice(["f32", "bf16", "bf16"])
    if op == "chunk":
        seqs = rng.choice([1, 1, 2, 3, 8, 16])
        tokens = _log(rng, 1, 8191 // seqs)
        c = _chunk(None, heads, kv, kind, tokens, _log(rng, 1, 32768 // seqs), seqs, page, rng.random() < 0.5,
                   window=rng.choice([0, 0, 0, _log(rng, 16, 4096)]), docs=rng.choice([0, 0, 0, 2, 5]), prefix=rng.choice([0, 0, 0, 1]),
                   cap=rng.choice([0.0, 0.0, 30.0]), bias=rng.choice([0.0, 0.0, 0.0, 8.0]))
        while work(c)["flops"] > 1.0e12 or _HEADS[heads][0] * seqs * c["tokens"] * (c["rows"] + c["tokens"]) > 4.3e9:
            big = "rows" if c["rows"] > c["tokens"] else "tokens"
            c[big] = c[big] * 4 // 5
        return c
    if op == "weights":
        seqs = rng.choice([1, 2, 3, 8, 16])
        tokens = rng.choice([1, 1, 2, 8, 16, 31, 32, 64, 200])
        return _weights(None, heads, kv, kind, tokens, _log(rng, 16, min(32768, (131072 if tokens < 64 else 32768) // seqs)), seqs, page,
                        rng.random() < 0.5, rng.choice([1.0, 0.9]), rng.choice([0, 0, 0, 1024]), rng.choice([0.0, 0.0, 30.0]))
    if op == "evict":
        seqs = rng.choice([1, 2, 5, 16, 32])
        rows = _log(rng, 32, 48000 // seqs)
        keep = rng.choice([rows - 1, rows - 8, rows // 2, rows // 3, rows // 8])
        return _evict(None, heads, kv, rng.choice([2, 4, 8]), page, rows, max(1, keep), seqs, rng.choice([0, 4]), rng.choice([0, 8, 64]),
                      rng.random() < 0.5)
    seqs = rng.choice([1, 1, 2, 5, 8, 16, 32])
    tokens = rng.choice([1, 2, 4, 6, 8, 16, 25, 33, 64])
    mode = rng.choice(["greedy", "target", "target", "draft", "draft"])
    return _verify(None, rng.choice(["f32", "bf16"]), _log(rng, 1000, min(160000, 33000000 // (seqs * tokens))), tokens, seqs, mode,
                   mode == "draft" or rng.random() < 0.3, rng.random() < 0.4)


def _lengths(c):
    """Rows that each sequence holds before the call, and its new tokens: of the case alone."""
    n, rows, t = c["seqs"], c.get("rows", 0), c["tokens"]
    if not c["ragged"]:
        return [rows] * n, [t] * n
    frac = [(0.381966 * b) % 1.0 for b in range(n)]
    held = [int(rows * math.exp(-4.0 * f)) for f in frac]
    return held, [max(1, int(t * (1.0 - 0.5 * ((0.7549 * b) % 1.0)))) for b in range(n)]


def _firsts(c, r, t):
    """The first row of the document that each new token belongs to: `docs` of them over rows [0, r + t)."""
    if not c["docs"]:
        return [0] * t
    cuts = [int((r + t) * ((k + 0.37) / (c["docs"] + 0.37))) for k in range(1, c["docs"])]
    return [max([0] + [x for x in cuts if x <= r + i]) for i in range(t)]


def _ranges(c):
    """For each sequence its rows, new tokens, and the [first, last) rows that each token sees."""
    for r, t in zip(*_lengths(c)):
        first = _firsts(c, r, t)
        pre = (r + t) // 2 if c["prefix"] else 0
        lo = [max(first[i], r + i + 1 - c["window"] if c["window"] else 0, 0) for i in range(t)]
        yield r, t, lo, [max(r + i + 1, pre) for i in range(t)]


def _evict_rows(c):
    """Rows and budget of each sequence."""
    rows = [max(2, c["rows"] - (b * 7) % max(1, c["rows"] // 4)) for b in range(c["seqs"])]
    return rows, [max(1, r - (c["rows"] - c["keep"])) if c["rows"] - c["keep"] < 16 else max(1, r * c["keep"] // c["rows"]) for r in rows]


def work(c):
    if c["op"] in ("chunk", "weights"):
        H, Hkv, D = _HEADS[c["heads"]]
        es, rec = _ELEM[c["type"]], _record(c["kv"], D)
        n = rows = seen = 0
        for r, t, lo, hi in _ranges(c):
            n += t
            rows += r + t - min(lo)
            seen += sum(b - a for a, b in zip(lo, hi))
        if c["op"] == "chunk":
            return {"bytes": 2 * n * H * D * es + 2 * rows * Hkv * rec, "flops": 4 * H * D * seen}
        return {"bytes": n * H * (D * es + 4) + rows * (Hkv * rec + 8), "flops": 2 * H * D * seen}
    if c["op"] == "evict":
        H, Hkv, D = _HEADS[c["heads"]]
        moved = total = 0
        for n, k in zip(*_evict_rows(c)):
            moved += round(k * (n - k) / n)
            total += n
        return {"bytes": 8 * total + 2 * moved * (2 * c["layers"] * Hkv * _record(c["kv"], D) + 8), "flops": 0}
    n = sum(_lengths(c)[1])
    rows = n + (c["seqs"] if c["mode"] == "draft" else 0)
    return {"bytes": rows * c["vocab"] * _ELEM[c["type"]], "flops": 4 * rows * c["vocab"]}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _store(x, kv):
    """float32 [..., D] as records of a cache type, uint8 [..., record]."""
    if kv not in ("q8_0", "q4_0"):
        return x.to(_TORCH[kv]).view(torch.uint8)
    b = x.reshape(*x.shape[:-1], -1, 32)
    if kv == "q8_0":
        d = b.abs().amax(-1, keepdim=True) / 127.0
        q = torch.round(b / d.clamp_min(1e-30)).clamp(-127, 127).to(torch.int8).view(torch.uint8)
    else:
        d = b.gather(-1, b.abs().argmax(-1, keepdim=True)) / -8.0
        n = torch.floor(b / d + 8.5).clamp(0, 15).to(torch.uint8)
        q = n[..., :16] | (n[..., 16:] << 4)
    return torch.cat([d.half().view(torch.uint8), q], -1).reshape(*x.shape[:-1], -1)


def _load(raw, kv, to):
    """Records uint8 [..., record] as their values [..., D] in the type `to`."""
    if kv not in ("q8_0", "q4_0"):
        return raw.view(_TORCH[kv]).to(to)
    b = raw.reshape(*raw.shape[:-1], -1, _ELEM[kv])
    d = b[..., :2].contiguous().view(torch.float16).to(to)
    q = b[..., 2:]
    v = q.contiguous().view(torch.int8).to(to) if kv == "q8_0" else torch.cat([q & 15, q >> 4], -1).to(to) - 8
    return (v * d).reshape(*raw.shape[:-1], -1)


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(int(seed))
    s = {"c": dict(case)}
    {"chunk": _prepare_attention, "weights": _prepare_attention, "evict": _prepare_evict, "verify": _prepare_verify}[case["op"]](s, g, int(seed))
    if own:
        _bind(s)
    return s


def _prepare_attention(s, g, seed):
    c = s["c"]
    H, Hkv, D = s["heads"] = _HEADS[c["heads"]]
    P, kv, B, T = c["page"], c["kv"], c["seqs"], c["tokens"]
    rec = _record(kv, D)

    def rand(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    def pool(n_pages):
        x = torch.empty((n_pages, P, Hkv, rec), dtype=torch.uint8, device="cuda")
        step = max(1, (1 << 25) // (P * Hkv * D))
        for i in range(0, n_pages, step):
            x[i:i + step] = _store(rand(min(step, n_pages - i), P, Hkv, D), kv)
        return x

    held, new = _lengths(c)
    need = [_cdiv(r + t, P) for r, t in zip(held, new)]
    n_pages = sum(need) + 3
    ids = torch.randperm(n_pages, generator=g, device="cuda").int()
    s["table"] = torch.full((B, max(need)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(need):
        s["table"][b, :n] = ids[at:at + n]
        at += n
    s["rows"], s["n_tok"] = _i32(held), _i32(new)
    s["first"] = None
    if c["docs"]:
        s["first"] = _i32([_firsts(c, r, t) + [0] * (T - t) for r, t in zip(held, new)])
    s["prefix"] = _i32([(r + t) // 2 for r, t in zip(held, new)]) if c["prefix"] else None
    s["q"] = (rand(B, T, H, D) * 1.3).to(_TORCH[c["type"]])
    s["K"] = pool(n_pages)
    if c["op"] == "chunk":
        s["V"] = pool(n_pages)
        s["out"] = torch.zeros((B, T, H, D), dtype=_TORCH[c["type"]], device="cuda")
        s["lse"] = torch.zeros((B, T, H), device="cuda") if c["type"] == "f32" else None
    else:
        s["V"] = s["K"]  # (not read)
        x, m, z = _scores(s)
        s["lse"] = (m + z.log())[..., 0].permute(0, 3, 1, 2).flatten(2, 3).contiguous()
        del x, m, z
        cols = max(r + t for r, t in zip(held, new)) + 5
        s["scores"] = rand(B, cols).exp_()
        s["scores_out"] = torch.zeros((B, cols), device="cuda")


def _prepare_evict(s, g, seed):
    c = s["c"]
    H, Hkv, D = s["heads"] = _HEADS[c["heads"]]
    P, rec, B = c["page"], _record(c["kv"], D), c["seqs"]
    rows, keep = _evict_rows(c)
    need = [_cdiv(r, P) for r in rows]
    stay = [_cdiv(k, P) for k in keep]
    # pages of what stays in any order; behind them, rising, those that a call gives back and the next takes again
    ids = torch.randperm(sum(stay), generator=g, device="cuda").int()
    s["table"] = torch.full((B, max(need)), -1, dtype=torch.int32, device="cuda")
    at, behind = 0, sum(stay)
    for b in range(B):
        s["table"][b, :stay[b]] = ids[at:at + stay[b]]
        at += stay[b]
        s["table"][b, stay[b]:need[b]] = torch.arange(behind, behind + need[b] - stay[b], device="cuda")
        behind += need[b] - stay[b]
    s["refs"] = torch.zeros(behind + 4, dtype=torch.int32, device="cuda")
    s["refs"][:behind] = 1
    s["rows"], s["keep"] = _i32(rows), _i32(keep)
    cols = max(rows) + 3
    # accumulated weights: of all magnitudes, many the same, rows that nothing has looked at
    x = torch.randn((B, cols), generator=g, device="cuda").mul_(2.0).exp_()
    x = torch.where(torch.rand((B, cols), generator=g, device="cuda") < 0.3, (x * 8).floor() / 8, x)
    s["scores"] = torch.where(torch.rand((B, cols), generator=g, device="cuda") < 0.1, torch.zeros_like(x), x)
    pos = torch.arange(cols, device="cuda", dtype=torch.int32).repeat(B, 1)
    if c["moved"]:  # rows that earlier evictions put in others' places
        pos = torch.rand((B, cols), generator=g, device="cuda").argsort(-1).int()
    s["pos"] = pos.contiguous()
    s["scores_out"], s["pos_out"] = torch.zeros_like(s["scores"]), torch.zeros_like(s["pos"])
    s["rows_out"], s["got"] = torch.zeros_like(s["rows"]), torch.zeros_like(s["rows"])
    shape = (2 * c["layers"], behind + 4, P, Hkv, rec)
    words = math.prod(shape) // 8
    s["pools"] = torch.randint(-2**62, 2**62, (words,), generator=g, device="cuda").view(torch.uint8).reshape(shape)


def _prepare_verify(s, g, seed):
    c = s["c"]
    B, T, V = c["seqs"], c["tokens"], c["vocab"]
    dt = _TORCH[c["type"]]
    plan = random.Random(seed)
    # a target that is sure of some tokens and unsure of others
    sharp = torch.rand((B, T, 1), generator=g, device="cuda") * 3.0 + 1.0
    x = torch.randn((B, T, V), generator=g, device="cuda").mul_(sharp)
    s["logits"] = x.to(dt)
    s["parents"] = None
    up = [[i - 1 for i in range(T)] for _ in range(B)]
    if not c["chain"]:
        up = [[-1] + [plan.randint(max(0, i - 6), i - 1) for i in range(1, T)] for _ in range(B)]
        s["parents"] = _i32(up)
    s["n_tok"] = _i32(_lengths({**c, "rows": 0})[1])
    s["temperature"] = torch.rand(B, generator=g, device="cuda") * 0.6 + 0.6
    if c["mode"] == "greedy":
        s["temperature"].zero_()
    s["uniform"] = torch.rand((B, T + 1), generator=g, device="cuda")
    s["draft"] = None
    up = _i32(up).long()
    if c["mode"] == "draft":
        # a draft that agrees with the target to some degree; its tokens are drawn from it
        y = x.div_(s["temperature"][:, None, None]).add_(torch.randn((B, T, V), generator=g, device="cuda"), alpha=0.7)
        q = torch.softmax(y, -1)
        s["draft"] = q.to(dt)
        drawn = torch.multinomial(q.view(B * T, V), 1, generator=g).view(B, T)
        s["tokens"] = drawn.roll(1, 1).int().contiguous()
    else:
        # the k-th child of a token is the k-th most likely token after it, now and then another one
        i = torch.arange(T, device="cuda")
        rank = ((up[:, :, None] == up[:, None, :]) & (i[:, None] > i)).sum(-1)
        top = s["logits"].float().topk(min(8, V), -1).indices
        best = top[torch.arange(B, device="cuda")[:, None], up.clamp(min=0), rank.clamp(max=top.shape[-1] - 1)]
        other = torch.randint(0, V, (B, T), generator=g, device="cuda")
        s["tokens"] = torch.where(torch.rand((B, T), generator=g, device="cuda") < 0.8, best, other).int().contiguous()
    s["path"] = torch.zeros((B, T), dtype=torch.int32, device="cuda")
    s["n_path"], s["next"] = (torch.zeros(B, dtype=torch.int32, device="cuda") for _ in range(2))
    s["logp"] = torch.zeros((B, T + 1), device="cuda")


# ---------------------------------------------------------------------------
# the library's calls: descriptors and workspace filled once, as a program does
# ---------------------------------------------------------------------------

def _library():
    pkg = pathlib.Path(__file__).resolve().parents[1] / "xllama-qwen35-xbox_amd"
    if str(pkg) not in sys.path:
        sys.path.insert(0, str(pkg))
    import xqattn
    return xqattn


def _ptr(t):
    return None if t is None else t.data_ptr()


def _bind(s):
    xq = _library()
    lib, c = xq.load(), s["c"]
    s["keep_alive"] = keep = []

    def tensor(typ, ne, nb, t):
        keep.append(xq.DevTensor(typ, ne, nb, t).desc())
        return ctypes.byref(keep[-1])

    def plane(t):
        H, Hkv, D = s["heads"]
        rec = _record(c["kv"], D)
        return xq.DevTensor(_TYPES[c["kv"]], (D, c["page"], Hkv, t.shape[0]), (_ELEM[c["kv"]], Hkv * rec, rec, c["page"] * Hkv * rec), t).desc()

    def space(query, *args):
        n = ctypes.c_size_t(0)
        st = query(*args, ctypes.byref(n))
        if st:
            raise RuntimeError("%s: %s" % (st, lib.xq_last_error().decode()))
        keep.append(torch.empty(n.value + 256, dtype=torch.uint8, device="cuda"))
        return keep[-1].data_ptr() + -keep[-1].data_ptr() % 256, n.value

    if c["op"] in ("chunk", "weights"):
        H, Hkv, D = s["heads"]
        B, T, es = c["seqs"], c["tokens"], _ELEM[c["type"]]
        q = tensor(_TYPES[c["type"]], (D, T, H, B), (es, H * D * es, D * es, T * H * D * es), s["q"])
        cache = xq.XqKvPages()
        cache.k, cache.v = plane(s["K"]), plane(s["V"])
        cache.table, cache.rows = _ptr(s["table"]), _ptr(s["rows"])
        cache.n_seq, cache.table_cols = s["table"].shape
        p = xq.chunk_params(1.0 / math.sqrt(D), window=c["window"], logit_softcap=c["cap"], max_bias=c["bias"])
        keep += [cache, p]
        cache, p = ctypes.byref(cache), ctypes.byref(p)
        masks = (_ptr(s["first"]), _ptr(s["prefix"]), _ptr(s["n_tok"]))
        if c["op"] == "chunk":
            out = tensor(_TYPES[c["type"]], (D, H, T, B), (es, D * es, H * D * es, T * H * D * es), s["out"])
            s["calls"] = [(lib.xq_fa_chunk, (q, cache, p, *masks, out, _ptr(s["lse"]), *space(lib.xq_fa_chunk_workspace, q, cache, out)))]
        else:
            s["calls"] = [(lib.xq_kv_weights, (q, cache, p, *masks, _ptr(s["lse"]), _ptr(s["scores"]), _ptr(s["scores_out"]),
                                               s["scores"].shape[1], c["decay"], 1, *space(lib.xq_kv_weights_workspace, q, cache)))]
    elif c["op"] == "evict":
        planes = s["pools"].shape[0]
        pools = (xq.XqTensor * planes)(*[plane(s["pools"][i]) for i in range(planes)])
        keep.append(pools)
        B, cols = s["table"].shape
        s["calls"] = [
            # the rows that the sequences hold have pages: those that the last pass gave back are taken again
            (lib.xq_kv_pages_reserve, (_ptr(s["table"]), _ptr(s["refs"]), B, cols, s["refs"].numel(), c["page"], _ptr(s["rows"]),
                                       _ptr(s["got"]), *space(lib.xq_kv_pages_reserve_workspace, B, s["refs"].numel()))),
            (lib.xq_kv_pages_evict, (pools, planes, _ptr(s["table"]), _ptr(s["rows"]), _ptr(s["refs"]), B, cols, _ptr(s["keep"]),
                                     c["first"], c["last"], _ptr(s["scores"]), _ptr(s["pos"]), s["scores"].shape[1],
                                     _ptr(s["scores_out"]), _ptr(s["pos_out"]), _ptr(s["rows_out"]),
                                     *space(lib.xq_kv_pages_evict_workspace, B, s["scores"].shape[1])))]
    else:
        B, T, V = s["logits"].shape
        es = _ELEM[c["type"]]
        ne, nb = (V, T, B, 1), (es, V * es, T * V * es, B * T * V * es)
        logits = tensor(_TYPES[c["type"]], ne, nb, s["logits"])
        draft = None if s["draft"] is None else tensor(_TYPES[c["type"]], ne, nb, s["draft"])
        s["calls"] = [(lib.xq_verify_tokens, (logits, draft, _ptr(s["tokens"]), _ptr(s["parents"]), _ptr(s["n_tok"]), _ptr(s["temperature"]),
                                              _ptr(s["uniform"]), _ptr(s["path"]), _ptr(s["n_path"]), _ptr(s["next"]), _ptr(s["logp"]),
                                              *space(lib.xq_verify_tokens_workspace, logits)))]


def _do(call):
    fn, args = call
    st = fn(*args, torch.cuda.current_stream().cuda_stream)
    if st:
        raise RuntimeError("%s: %s" % (st, _library().load().xq_last_error().decode()))


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(s):
    c = s["c"]
    if own:
        _do(s["calls"][0])
        if c["op"] == "evict":
            _do(s["calls"][1])
    elif c["op"] == "chunk":
        _plain_chunk(s)
    elif c["op"] == "weights":
        _plain_weights(s)
    elif c["op"] == "evict":
        _plain_evict(s)
    else:
        _plain_verify(s)
    if c["op"] == "chunk":
        return {"out": s["out"], "lse": s["lse"]}
    if c["op"] == "weights":
        return {"scores": s["scores_out"]}
    if c["op"] == "evict":
        return {"pools": s["pools"].view(-1).view(torch.int64), "table": s["table"], "refs": s["refs"], "rows": s["rows_out"],
                "scores": s["scores_out"].view(torch.int32), "positions": s["pos_out"]}
    return {"path": s["path"], "n_path": s["n_path"], "next": s["next"], "logp": s["logp"]}


def _slopes(H, bias):
    """ALiBi slopes of the heads."""
    n = 2 ** int(math.log2(H))
    h = torch.arange(H, device="cuda", dtype=torch.float64)
    return torch.where(h < n, 2.0 ** (-bias / n * (h + 1)), 2.0 ** (-bias / 2 / n * (2 * (h - n) + 1)))


def _scores(s):
    """Masked scores [B, Hkv, G, T, rows] less their maxima, exponentiated; the maxima; the sums."""
    c = s["c"]
    (H, Hkv, D), B, T = s["heads"], c["seqs"], c["tokens"]
    G = H // Hkv
    k = _load(s["K"][s["table"].clamp(min=0).long()].flatten(1, 2), c["kv"], torch.float32).transpose(1, 2)  # [B, Hkv, rows, D]
    q = s["q"].float().unflatten(2, (Hkv, G)).permute(0, 2, 3, 1, 4).reshape(B, Hkv, G * T, D)
    x = (q @ k.transpose(2, 3)).mul_(1.0 / math.sqrt(D)).unflatten(2, (G, T))
    del q, k
    if c["cap"]:
        x.div_(c["cap"]).tanh_().mul_(c["cap"])
    r = torch.arange(x.shape[-1], device="cuda")
    p = s["rows"][:, None] + torch.arange(T, device="cuda")
    if c["bias"]:
        x.add_(_slopes(H, c["bias"]).float().view(1, Hkv, G, 1, 1) * (r - p[..., None]).float()[:, None, None])
    hi = p + 1 if s["prefix"] is None else torch.maximum(p + 1, s["prefix"][:, None])
    lo = torch.zeros_like(p) if not c["window"] else p + 1 - c["window"]
    if s["first"] is not None:
        lo = torch.maximum(lo, s["first"])
    seen = (r >= lo[..., None]) & (r < hi[..., None]) & (r < (s["rows"] + s["n_tok"])[:, None, None])
    x.masked_fill_(~seen[:, None, None], -math.inf)
    m = x.amax(-1, keepdim=True).clamp(min=-3e38)
    x.sub_(m).exp_()
    return x, m, x.sum(-1, keepdim=True)


def _plain_chunk(s):
    c, T = s["c"], s["c"]["tokens"]
    x, m, z = _scores(s)
    v = _load(s["V"][s["table"].clamp(min=0).long()].flatten(1, 2), c["kv"], torch.float32).transpose(1, 2)
    o = (x.flatten(2, 3) @ v).unflatten(2, (x.shape[2], T)) / z
    live = torch.arange(T, device="cuda") < s["n_tok"][:, None]
    o = o.permute(0, 3, 1, 2, 4).flatten(2, 3)
    s["out"].copy_(torch.where(live[..., None, None], o.to(s["out"].dtype), s["out"]))
    if s["lse"] is not None:
        lse = (m + z.log())[..., 0].permute(0, 3, 1, 2).flatten(2, 3)
        s["lse"].copy_(torch.where(live[..., None], lse, s["lse"]))


def _plain_weights(s):
    c, T = s["c"], s["c"]["tokens"]
    (H, Hkv, D), B = s["heads"], c["seqs"]
    x, m, _ = _scores(s)
    lse = s["lse"].unflatten(2, (Hkv, H // Hkv)).permute(0, 2, 3, 1)[..., None]
    live = (torch.arange(T, device="cuda") < s["n_tok"][:, None])[:, None, None, :, None]
    w = x.mul_(torch.where(live, (m - lse).exp(), torch.zeros_like(m))).sum((1, 2, 3))
    cols = s["scores"].shape[1]
    w = torch.nn.functional.pad(w, (0, max(0, cols - w.shape[1])))[:, :cols]
    r = torch.arange(cols, device="cuda")
    old = torch.where(r < s["rows"][:, None], s["scores"] * c["decay"], torch.zeros_like(s["scores"]))
    s["scores_out"].copy_(torch.where(r < (s["rows"] + s["n_tok"])[:, None], old + w, s["scores_out"]))


def _plain_evict(s):
    c, P = s["c"], s["c"]["page"]
    table, refs, n, k = s["table"], s["refs"], s["rows"][:, None], s["keep"][:, None]
    # the rows' pages
    col = torch.arange(table.shape[1], device="cuda")
    missing = (col < (n + P - 1) // P) & (table < 0)
    free = (refs == 0).nonzero()[:, 0][:missing.sum()]
    table[missing] = free.int()
    refs[free] = 1
    # which rows stay: protected ones, then by score, then by index
    r = torch.arange(s["scores"].shape[1], device="cuda")
    held = r < n
    newest = torch.where(held, s["pos"], torch.zeros_like(s["pos"])).amax(-1, keepdim=True)
    safe = held & ((s["pos"] < c["first"]) | (newest - s["pos"] < c["last"]))
    order = torch.where(held, s["scores"], torch.full_like(s["scores"], -1.0)).sort(dim=-1, descending=True, stable=True).indices
    again = safe.gather(1, order).int().sort(dim=-1, descending=True, stable=True).indices
    order = order.gather(1, again)
    stays = torch.zeros_like(held).scatter_(1, order, r < k) & held
    s["scores_out"].copy_(torch.where(r < k, s["scores"], s["scores_out"]))
    s["pos_out"].copy_(torch.where(r < k, s["pos"], s["pos_out"]))
    b, hole = ((r < k) & ~stays).nonzero(as_tuple=True)
    _, from_ = ((r >= k) & stays).nonzero(as_tuple=True)
    s["scores_out"][b, hole] = s["scores"][b, from_]
    s["pos_out"][b, hole] = s["pos"][b, from_]
    flat = s["pools"].flatten(1, 2).view(torch.int64 if s["pools"].shape[-1] % 8 == 0 else torch.int16)
    src, dst = (table[b, x // P].long() * P + x % P for x in (from_, hole))
    flat[:, dst] = flat[:, src]
    s["rows_out"].copy_(s["keep"])
    gone = (col >= (k + P - 1) // P) & (table >= 0)
    refs[table[gone].long()] = 0
    table[gone] = -1


def _plain_verify(s):
    c, T = s["c"], s["c"]["tokens"]
    B, V = c["seqs"], c["vocab"]
    i = torch.arange(T, device="cuda")
    seq = torch.arange(B, device="cuda")
    tok, u = s["tokens"].long(), s["uniform"].double()
    up = (i - 1).expand(B, T) if s["parents"] is None else s["parents"].long()
    live = i < s["n_tok"][:, None]
    heat = torch.where(s["temperature"] > 0, s["temperature"], torch.ones_like(s["temperature"])).double()
    logp = torch.log_softmax(s["logits"].double() / heat[:, None, None], -1)
    lx = logp[seq[:, None], up.clamp(min=0), tok]
    siblings = (up[:, :, None] == up[:, None, :]) & (i[:, None] > i)  # [.., c, c']: c' an earlier child of the same token
    twice = (siblings & (tok[:, :, None] == tok[:, None, :])).any(-1)
    if c["mode"] == "greedy":
        x = s["logits"]
        best = torch.where(x == x.amax(-1, keepdim=True), torch.arange(V, device="cuda"), V).amin(-1)
        ok = tok == best.gather(1, up.clamp(min=0))
    elif c["mode"] == "draft":
        ok = u[:, :T] * s["draft"][seq[:, None], up.clamp(min=0), tok].double() < lx.exp()
    else:
        px = torch.where(twice, torch.zeros_like(lx), lx.exp())
        left = 1.0 - (siblings.double() * px[:, None, :]).sum(-1)
        ok = u[:, :T] * left < px
    ok &= live & (up >= 0)
    ok[:, 0] = live[:, 0]
    chosen = ok & ~(siblings & ok[:, None, :]).any(-1)
    # on the path: chosen, and so is every token above
    above = ((up[..., None] == i) | (i[:, None] == i)).float()
    for _ in range(max(1, (T - 1).bit_length())):
        above = (above @ above > 0).float()
    on = chosen & ~((above > 0) & ~chosen[:, None, :]).any(-1)
    n = on.sum(-1)
    s["n_path"].copy_(n)
    s["path"].copy_(torch.where(i < n[:, None], torch.where(on, i, T).sort(-1).values, -1))
    at = torch.where(on, i, -1).amax(-1).clamp(min=0)
    if c["mode"] == "greedy":
        nxt = best[seq, at]
    else:
        w = logp[seq, at].exp()
        kids = live & (up == at[:, None])
        if c["mode"] == "draft":
            w = torch.where(kids.any(-1, keepdim=True), (w - s["draft"][seq, at].double()).clamp(min=0), w)
        else:
            w = w * torch.ones((B, V + 1), dtype=w.dtype, device="cuda").scatter_(1, torch.where(kids, tok, V), 0.0)[:, :V]
        run_ = w.cumsum(-1)
        nxt = (run_ <= u[:, T:] * run_[:, -1:]).sum(-1).clamp(max=V - 1)
    s["next"].copy_(torch.where(n > 0, nxt, -1))
    last = torch.where(n > 0, logp[seq, at, nxt], 0.0)
    s["logp"].copy_(torch.cat([torch.where(live & (up >= 0), lx, 0.0), last[:, None]], -1))


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------

def exact(case, seed):
    if case["op"] == "evict":
        return None  # moves and counts: whole numbers
    if case["op"] == "verify":
        return _exact_verify(prepare(case, seed))
    H, Hkv, D = _HEADS[case["heads"]]
    if sum(t * (r + t) for r, t in zip(*_lengths(case))) * H * D > 1.2e12:
        return None
    s = prepare(case, seed)
    return _exact_chunk(s) if case["op"] == "chunk" else _exact_weights(s)


def _exact_rows(s):
    """For each sequence and query head: its number, the head, its tokens, and the scores [t, rows] in 64 bits, -inf where nothing is seen."""
    c = s["c"]
    (H, Hkv, D), P = s["heads"], c["page"]
    slope = _slopes(H, c["bias"]).tolist() if c["bias"] else None
    for b, (r, t, lo, hi) in enumerate(_ranges(c)):
        n = r + t
        pages = s["table"][b, :_cdiv(n, P)].long()
        row = torch.arange(n, device="cuda")
        seen = (row >= torch.tensor(lo, device="cuda")[:, None]) & (row < torch.tensor(hi, device="cuda")[:, None])
        far = (row - torch.arange(r, n, device="cuda")[:, None]).double() if slope else None
        for h in range(Hkv):
            k = _load(s["K"][pages, :, h].flatten(0, 1)[:n], c["kv"], torch.float64)
            for e in range(h * (H // Hkv), (h + 1) * (H // Hkv)):
                x = s["q"][b, :t, e].double() @ k.T / math.sqrt(D)
                if c["cap"]:
                    x = torch.tanh(x / c["cap"]) * c["cap"]
                if slope:
                    x = x + far * slope[e]
                yield b, e, t, pages, torch.where(seen, x, -math.inf)


def _exact_chunk(s):
    c, (H, Hkv, D) = s["c"], s["heads"]
    out = s["out"].double()
    lse = None if s["lse"] is None else s["lse"].double()
    for b, e, t, pages, x in _exact_rows(s):
        z = torch.logsumexp(x, -1)
        v = _load(s["V"][pages, :, e // (H // Hkv)].flatten(0, 1)[:x.shape[1]], c["kv"], torch.float64)
        out[b, :t, e] = torch.exp(x - z[:, None]) @ v
        if lse is not None:
            lse[b, :t, e] = z
    return {"out": out, "lse": lse}


def _exact_weights(s):
    c = s["c"]
    out = s["scores_out"].double()
    held = s["rows"].tolist()
    for b, r in enumerate(held):
        out[b, :r] = s["scores"][b, :r].double() * c["decay"]
    for b, e, t, pages, x in _exact_rows(s):
        out[b, :x.shape[1]] += torch.exp(x - s["lse"][b, :t, e].double()[:, None]).sum(0)
    return {"scores": out}


def _exact_verify(s):
    """The logarithms of the tokens' probabilities; the tokens are whole numbers, and the next one's follows from them."""
    c = s["c"]
    up = [[j - 1 for j in range(c["tokens"])]] * c["seqs"] if s["parents"] is None else s["parents"].tolist()
    tok, heat = s["tokens"].tolist(), s["temperature"].tolist()
    _plain_verify(s)
    nxt, path, n_path = s["next"].tolist(), s["path"].tolist(), s["n_path"].tolist()
    out = torch.zeros((c["seqs"], c["tokens"] + 1), dtype=torch.float64)
    for b, n in enumerate(s["n_tok"].tolist()):
        x = s["logits"][b].double() / (heat[b] if heat[b] > 0 else 1.0)
        x = (x - x.logsumexp(-1, keepdim=True)).cpu()
        for j in range(1, n):
            out[b, j] = x[up[b][j], tok[b][j]]
        out[b, -1] = x[path[b][n_path[b] - 1], nxt[b]]
    return {"path": None, "n_path": None, "next": None, "logp": out}
