"""The paged-cache operators as measurable cases: plain torch forms beside the library's calls.

Three operators of one serving step over a KV cache that is kept in pages:

* ``rope``   ``xq_qk_norm_rope``: each head's RMS norm and position rotation of queries and
             keys, K and V stored into the pages of their sequence in the same pass;
* ``tree``   ``xq_fa_tree``: attention of a tree of drafted tokens (of one token: a decode
             step) over the paged cache;
* ``pages``  ``xq_kv_pages_*``: the accepted path of a tree moved to the front (``compact``),
             losing beams released and winning ones forked (``beams``), pages copied to
             other places (``copy``).

Head shapes are the repository's own (24 query heads over 4 KV heads at head dim 256, 16 over 8
and 32 over 8 at 128). A case's lengths follow from the case alone; its values come from the
seed. Where ``own`` is false, ``run`` computes the operator from elementary torch operations in
32 bits (angles in 64). Caches that ``rope`` fills are f16, bf16 or e5m2 here: a q8_0 or q4_0 code
next to a border may be rounded either way by 32-bit sums of another order.
"""
import ctypes
import math
import pathlib
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

def _rope(name, heads, kv, kind, tokens, seqs, n_rot, page, rows, ragged=False, mode="halves"):
    c = {"op": "rope", "heads": heads, "kv": kv, "type": kind, "tokens": tokens, "seqs": seqs, "n_rot": n_rot,
         "page": page, "rows": rows, "ragged": ragged, "mode": mode}
    return {"name": name, **c} if name else c


def _tree(name, heads, kv, kind, tokens, rows, seqs, page, ragged=False, chain=False):
    c = {"op": "tree", "heads": heads, "kv": kv, "type": kind, "tokens": tokens, "rows": rows, "seqs": seqs,
         "page": page, "ragged": ragged, "chain": chain}
    return {"name": name, **c} if name else c


def _pages(name, part, heads, kv, layers, page, rows, seqs, tokens=0, accepted=0, count=0):
    c = {"op": "pages", "part": part, "heads": heads, "kv": kv, "layers": layers, "page": page, "rows": rows,
         "seqs": seqs, "tokens": tokens, "accepted": accepted, "count": count}
    return {"name": name, **c} if name else c


def listed():
    return [
        # the decode step of one user, f32 rows as a ggml graph hands them over: latency
        _rope("rope_decode_f32", "24/4/256", "f16", "f32", 1, 1, 64, 16, 1000),
        # eight users' trees of up to 25 drafted tokens, ragged, fp8 cache
        _rope("rope_tree25_bf16_b8", "32/8/128", "e5m2", "bf16", 25, 8, 128, 16, 9001, ragged=True),
        # a prompt batch: two prompts of 4097 tokens, a quarter of each head rotated
        _rope("rope_prompt_bf16_4k_b2", "24/4/256", "f16", "bf16", 4097, 2, 64, 64, 0),
        # a chat that has just begun, one token: latency
        _tree("tree_decode_q8_377", "24/4/256", "q8_0", "f32", 1, 377, 1, 16),
        # a verify of four tokens in a row on one user's 4k context
        _tree("tree_chain4_f16_4k", "16/8/128", "f16", "f32", 4, 4097, 1, 16, chain=True),
        # a decode batch of 32 chats of all lengths, one token each, fp8 cache
        _tree("tree_decode_e5m2_b32", "16/8/128", "e5m2", "bf16", 1, 8000, 32, 64, ragged=True),
        # two agents' long contexts, 16 drafted tokens each, head dim 256
        _tree("tree16_q8_12k_b2", "24/4/256", "q8_0", "bf16", 16, 12289, 2, 32),
        # sixteen users of all lengths, trees of up to 25 tokens, 4-bit cache
        _tree("tree25_q4_16k_b16", "32/8/128", "q4_0", "bf16", 25, 16391, 16, 16, ragged=True),
        # the largest: four long contexts, 64 drafted tokens each
        _tree("tree64_f16_32k_b4", "32/8/128", "f16", "bf16", 64, 32768, 4, 64),
        # after a verify: the accepted path's rows of every attention layer moved to the front
        _pages("accept_f16_b8", "compact", "16/8/128", "f16", 8, 16, 2003, 8, tokens=25, accepted=5),
        # a beam search step: 16 losing beams released, 16 winners forked
        _pages("beams_q8_b32", "beams", "24/4/256", "q8_0", 16, 64, 1501, 32, count=16),
        # a cache put in order: 512 pages of 8 layers to other places
        _pages("copy_f16_512", "copy", "32/8/128", "f16", 8, 32, 0, 0, count=512),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "tree", "tree", "tree", "pages"])
    heads = rng.choice(sorted(_HEADS))
    page = rng.choice([16, 16, 32, 64, 128])
    if op == "rope":
        seqs = rng.choice([1, 1, 2, 3, 8, 17])
        n_rot = rng.choice([64, 128] if heads.endswith("128") else [64, 64, 128, 256])
        kind = rng.choice(["f32", "bf16"])
        return _rope(None, heads, rng.choice(["f16", "bf16", "e5m2"]), kind, _log(rng, 1, (8192 if kind == "bf16" else 4096) // seqs),
                     seqs, n_rot, page, _log(rng, 1, 20000), rng.random() < 0.5, rng.choice(["halves", "halves", "pairs"]))
    if op == "tree":
        seqs = rng.choice([1, 1, 2, 4, 7, 16, 32])
        tokens = rng.choice([1, 1, 2, 4, 7, 8, 16, 25, 33, 48, 64])
        rows = _log(rng, 16, min(49152, (131072 if heads.endswith("128") else 87381) // seqs))
        return _tree(None, heads, rng.choice(["f16", "q8_0", "q8_0", "q4_0", "e5m2"]), rng.choice(["f32", "bf16", "bf16"]),
                     tokens, rows, seqs, page, rng.random() < 0.5, rng.random() < 0.25)
    part = rng.choice(["compact", "beams", "copy"])
    kv = rng.choice(["f16", "q8_0", "q4_0", "e5m2"])
    if part == "compact":
        tokens = rng.randint(4, 64)
        return _pages(None, part, heads, kv, rng.choice([2, 4, 8]), page, _log(rng, 40, 2500), rng.randint(1, 16), tokens,
                      rng.randint(2, min(8, tokens)))
    if part == "beams":
        seqs = 2 * rng.randint(2, 16)
        return _pages(None, part, heads, kv, rng.choice([2, 4, 8]), page, _log(rng, 40, 2000), seqs, count=rng.randint(1, seqs // 2))
    return _pages(None, part, heads, kv, rng.choice([2, 4, 8]), page, 0, 0, count=_log(rng, 8, 8192 // page))


def _lengths(c):
    """Rows that each sequence holds before the call, and its new tokens: of the case alone."""
    n, rows, t = c["seqs"], c["rows"], c.get("tokens", 0)
    if not c.get("ragged"):
        return [rows] * n, [t] * n
    frac = [(0.381966 * b) % 1.0 for b in range(n)]
    held = [max(1, int(rows * math.exp(-4.0 * f))) for f in frac]
    return held, [max(1, int(t * (1.0 - 0.5 * ((0.7549 * b) % 1.0)))) for b in range(n)]


def _path(c):
    """The accepted path of a tree: rising indexes of drafted tokens."""
    a, t = c["accepted"], c["tokens"]
    return [j * (t - 1) // max(1, a - 1) for j in range(a)]


def _beam_rows(c):
    return [max(1, c["rows"] - 13 * b) for b in range(c["seqs"] // 2)]


def work(c):
    H, Hkv, D = _HEADS[c["heads"]]
    rec = _record(c["kv"], D)
    if c["op"] == "rope":
        es = _ELEM[c["type"]]
        n = sum(_lengths(c)[1])
        return {"bytes": n * (D * es * (2 * H + 2 * Hkv) + 2 * Hkv * rec), "flops": n * D * (10 * H + 10 * Hkv)}
    if c["op"] == "tree":
        es = _ELEM[c["type"]]
        held, new = _lengths(c)
        return {"bytes": sum(2 * Hkv * rec * (r + t) + 2 * H * D * es * t for r, t in zip(held, new)),
                "flops": sum(4 * H * D * t * (r + 0.5 * (t + 1)) for r, t in zip(held, new))}
    if c["part"] == "compact":
        moved = sum(p != j for j, p in enumerate(_path(c))) * c["seqs"]
        return {"bytes": 2 * 2 * c["layers"] * moved * Hkv * rec, "flops": 0}
    if c["part"] == "beams":
        part = [r % c["page"] for r in _beam_rows(c)]
        copied = sum(part[i % len(part)] for i in range(c["count"]))
        return {"bytes": 2 * 2 * c["layers"] * copied * Hkv * rec + 4 * c["count"] * 2 * _cdiv(c["rows"], c["page"]), "flops": 0}
    return {"bytes": 2 * 2 * c["layers"] * c["count"] * c["page"] * Hkv * rec, "flops": 0}


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


def _tables(g, need, cols, spare):
    """A page table whose sequences hold `need` pages each, in shuffled places of a pool with `spare` more."""
    n_pages = sum(need) + spare
    ids = torch.randperm(n_pages, generator=g, device="cuda").int()
    table = torch.full((len(need), cols), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = ids[at:at + n]
        at += n
    return table, n_pages


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _parents(g, B, T, chain):
    if chain:
        return torch.arange(-1, T - 1, dtype=torch.int32, device="cuda").repeat(B, 1)
    u = torch.rand((B, T), generator=g, device="cuda")
    i = torch.arange(T, device="cuda")
    return torch.where(i > 0, (u * i).floor(), torch.full_like(u, -1.0)).int()


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator("cuda").manual_seed(int(seed))
    H, Hkv, D = _HEADS[c["heads"]]
    P, kv = c["page"], c["kv"]
    rec = _record(kv, D)
    s = {"c": c, "H": H, "Hkv": Hkv, "D": D}

    def rand(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    def pool(n_pages):
        x = torch.empty((n_pages, P, Hkv, rec), dtype=torch.uint8, device="cuda")
        step = max(1, (1 << 25) // (P * Hkv * D))
        for i in range(0, n_pages, step):
            x[i:i + step] = _store(rand(min(step, n_pages - i), P, Hkv, D), kv)
        return x

    if c["op"] in ("rope", "tree"):
        held, new = _lengths(c)
        B, T = c["seqs"], c["tokens"]
        need = [_cdiv(r + t, P) for r, t in zip(held, new)]
        s["table"], n_pages = _tables(g, need, max(need), 3)
        s["rows"], s["n_tok"], s["B"], s["T"] = _i32(held), _i32(new), B, T
        dt = _TORCH[c["type"]]
        if c["op"] == "rope":
            # 24/4/256: a gate beside every query head, as the model's fused projection has it
            gate = 2 if D == 256 else 1
            x = (rand(B, T, (gate * H + 2 * Hkv) * D) * 1.5).to(dt)
            s["x"] = x
            s["q"] = x[..., :gate * H * D].unflatten(-1, (H, gate * D))[..., :D]
            s["k"] = x[..., gate * H * D:][..., :Hkv * D].unflatten(-1, (Hkv, D))
            s["v"] = x[..., (gate * H + Hkv) * D:].unflatten(-1, (Hkv, D))
            s["wq"], s["wk"] = 1.0 + 0.1 * rand(D), 1.0 + 0.1 * rand(D)
            depth = torch.arange(T, device="cuda", dtype=torch.int32)
            s["pos"] = (s["rows"][:, None] + 100000 * (int(seed) % 3) + depth).int().contiguous()
            s["out"] = torch.zeros((B, T, H, D), dtype=dt, device="cuda")
            zero = lambda: torch.zeros((n_pages, P, Hkv, rec), dtype=torch.uint8, device="cuda")  # noqa: E731
            s["K"], s["V"] = zero(), zero()
        else:
            s["q"] = rand(B, T, H, D).to(dt)
            s["parents"] = _parents(g, B, T, c["chain"])
            s["K"], s["V"] = pool(n_pages), pool(n_pages)
            s["out"] = torch.zeros((B, T, H, D), dtype=dt, device="cuda")
            s["lse"] = torch.zeros((B, T, H), device="cuda") if c["type"] == "f32" else None
    else:
        planes = 2 * c["layers"]
        if c["part"] == "compact":
            B = c["seqs"]
            held = [max(1, c["rows"] - 11 * b) for b in range(B)]
            need = [_cdiv(r + c["tokens"], P) for r in held]
            s["table"], n_pages = _tables(g, need, max(need), 3)
            s["rows"] = _i32(held)
            s["path"] = _i32([_path(c)] * B)
            s["n_path"] = _i32([len(_path(c))] * B)
            s["rows_out"] = torch.zeros_like(s["rows"])
        elif c["part"] == "beams":
            half, n = c["seqs"] // 2, c["count"]
            held = _beam_rows(c)
            need = [_cdiv(r, P) for r in held] + [0] * (c["seqs"] - half)
            s["table"], n_pages = _tables(g, need, max(need) + 1, n + 5)
            s["rows"] = _i32(held + [0] * (c["seqs"] - half))
            s["refs"] = torch.zeros(n_pages, dtype=torch.int32, device="cuda")
            s["refs"][s["table"][s["table"] >= 0].long()] = 1
            s["from"], s["to"] = _i32([i % half for i in range(n)]), _i32([half + i for i in range(n)])
            s["done"] = torch.zeros(n, dtype=torch.int32, device="cuda")
        else:
            n_pages = 2 * c["count"] + 5
            ids = torch.randperm(n_pages, generator=g, device="cuda").int()
            s["from"], s["to"] = ids[:c["count"]].contiguous(), ids[c["count"]:2 * c["count"]].contiguous()
        shape = (planes, n_pages, P, Hkv, rec)
        words = planes * n_pages * P * Hkv * rec // 8
        s["pools"] = torch.randint(-2**62, 2**62, (words,), generator=g, device="cuda").view(torch.uint8).reshape(shape)
    if own:
        _bind(s)
    return s


# ---------------------------------------------------------------------------
# the library's calls: descriptors and workspace filled once, as a program does
# ---------------------------------------------------------------------------

def _library():
    pkg = pathlib.Path(__file__).resolve().parents[1] / "xllama-qwen35-xbox_amd"
    if str(pkg) not in sys.path:
        sys.path.insert(0, str(pkg))
    import xqattn
    return xqattn


def _bind(s):
    xq = _library()
    lib, c, D, P = xq.load(), s["c"], s["D"], s["c"]["page"]
    kt, rec, Hkv = _TYPES[c["kv"]], _record(c["kv"], s["D"]), s["Hkv"]
    esz = _ELEM[c["kv"]]

    def ptr(t):
        return None if t is None else t.data_ptr()

    def tensor(typ, ne, nb, t):
        return xq.DevTensor(typ, ne, nb, t).desc()

    def plane(t):
        return tensor(kt, (D, P, Hkv, t.shape[0]), (esz, Hkv * rec, rec, P * Hkv * rec), t)

    def rows4(t):  # [B, T, heads, D] -> [D, T, heads, B]
        es = t.element_size()
        return tensor(_TYPES[c["type"]], (D, t.shape[1], t.shape[2], t.shape[0]),
                      (es, t.stride(1) * es, t.stride(2) * es, t.stride(0) * es), t)

    if c["op"] in ("rope", "tree"):
        cache = xq.XqKvPages()
        cache.k, cache.v = plane(s["K"]), plane(s["V"])
        cache.table, cache.rows = ptr(s["table"]), ptr(s["rows"])
        cache.n_seq, cache.table_cols = s["table"].shape
        if c["op"] == "rope":
            p = xq.rope_params(c["n_rot"], 1e7, mode=xq.ROPE_HALVES if c["mode"] == "halves" else xq.ROPE_PAIRS, eps=1e-6)
            keep = [rows4(s["q"]), rows4(s["k"]), rows4(s["v"]), p, rows4(s["out"]), cache]
            r = [ctypes.byref(x) for x in keep]
            s["call"] = (lib.xq_qk_norm_rope, (r[0], r[1], r[2], ptr(s["pos"]), ptr(s["n_tok"]), ptr(s["wq"]), ptr(s["wk"]), None,
                                               r[3], r[4], r[5]))
        else:
            o = s["out"]
            es = o.element_size()
            out = tensor(_TYPES[c["type"]], (D, s["H"], s["T"], s["B"]), (es, D * es, s["H"] * D * es, s["T"] * s["H"] * D * es), o)
            keep = [rows4(s["q"]), cache, out]
            r = [ctypes.byref(x) for x in keep]
            n = ctypes.c_size_t(0)
            assert lib.xq_fa_tree_workspace(r[0], r[1], r[2], ctypes.byref(n)) == 0, lib.xq_last_error()
            s["ws"] = torch.empty(n.value + 256, dtype=torch.uint8, device="cuda")
            at = s["ws"].data_ptr() + -s["ws"].data_ptr() % 256
            s["call"] = (lib.xq_fa_tree, (r[0], r[1], ptr(s["parents"]), ptr(s["n_tok"]), r[2], ptr(s["lse"]),
                                          1.0 / math.sqrt(D), at, n.value))
        s["keep"] = keep
        return
    planes = s["pools"].shape[0]
    pools = (xq.XqTensor * planes)(*[plane(s["pools"][i]) for i in range(planes)])
    s["keep"] = pools
    if c["part"] == "compact":
        s["call"] = (lib.xq_kv_pages_compact, (pools, planes, ptr(s["table"]), ptr(s["rows"]), s["table"].shape[0], s["table"].shape[1],
                                               ptr(s["path"]), ptr(s["n_path"]), s["path"].shape[1], ptr(s["rows_out"])))
    elif c["part"] == "beams":
        n_seq, cols = s["table"].shape
        n = ctypes.c_size_t(0)
        assert lib.xq_kv_pages_fork_workspace(c["count"], ctypes.byref(n)) == 0, lib.xq_last_error()
        s["ws"] = torch.empty(n.value + 256, dtype=torch.uint8, device="cuda")
        at = s["ws"].data_ptr() + -s["ws"].data_ptr() % 256
        s["release"] = (lib.xq_kv_pages_release, (ptr(s["table"]), ptr(s["rows"]), ptr(s["refs"]), n_seq, cols, s["refs"].numel(),
                                                  ptr(s["to"]), c["count"]))
        s["call"] = (lib.xq_kv_pages_fork, (pools, planes, ptr(s["table"]), ptr(s["rows"]), ptr(s["refs"]), n_seq, cols,
                                            ptr(s["from"]), ptr(s["to"]), c["count"], ptr(s["done"]), at, n.value))
    else:
        s["call"] = (lib.xq_kv_pages_copy, (pools, planes, ptr(s["from"]), ptr(s["to"]), c["count"]))


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
        if "release" in s:
            _do(s["release"])
        _do(s["call"])
    elif c["op"] == "rope":
        _plain_rope(s)
    elif c["op"] == "tree":
        _plain_tree(s)
    else:
        _plain_pages(s)
    if c["op"] == "rope":
        dt = _TORCH[c["kv"]]
        return {"q": s["out"], "k": s["K"].view(dt), "v": s["V"].view(dt)}
    if c["op"] == "tree":
        return {"out": s["out"], "lse": s["lse"]}
    pools = s["pools"].view(-1).view(torch.int64)
    if c["part"] == "compact":
        return {"pools": pools, "rows": s["rows_out"]}
    if c["part"] == "beams":
        return {"pools": pools, "table": s["table"], "rows": s["rows"], "refs": s["refs"], "done": s["done"]}
    return {"pools": pools}


def _slots(s):
    """Flat pool row of each new token, and which of them there are."""
    P = s["c"]["page"]
    i = torch.arange(s["T"], device="cuda")
    r = s["rows"][:, None].long() + i
    live = i < s["n_tok"][:, None]
    page = s["table"].gather(1, (r // P).clamp(max=s["table"].shape[1] - 1)).long()
    return page * P + r % P, live


def _plain_rope(s):
    c, D, n_rot = s["c"], s["D"], s["c"]["n_rot"]
    half = n_rot // 2
    f = 1e7 ** (torch.arange(half, device="cuda", dtype=torch.float64) * (-2.0 / n_rot))
    angle = s["pos"].double()[..., None, None] * f
    cos, sin = angle.cos().float(), angle.sin().float()

    def turn(x, w):
        x = x.float()
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w
        rot, rest = x[..., :n_rot], x[..., n_rot:]
        if c["mode"] == "halves":
            a, b = rot[..., :half], rot[..., half:]
            return torch.cat([a * cos - b * sin, a * sin + b * cos, rest], -1)
        a, b = rot[..., 0::2], rot[..., 1::2]
        return torch.cat([torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2), rest], -1)

    slot, live = _slots(s)
    q = turn(s["q"], s["wq"])
    s["out"].copy_(torch.where(live[..., None, None], q.to(s["out"].dtype), s["out"]))
    at = slot[live]
    dt = _TORCH[c["kv"]]
    for x, pool in ((turn(s["k"], s["wk"]), s["K"]), (s["v"].float(), s["V"])):
        x = x[live]
        x = x.half().to(dt) if c["kv"] == "e5m2" else x.to(dt)
        pool.view(-1, s["Hkv"], pool.shape[-1])[at] = x.view(torch.uint8)


def _seen(s, cols):
    """[B, T, cols] truth: the cache rows each token sees."""
    T, i = s["T"], torch.arange(s["T"], device="cuda")
    a = ((s["parents"][..., None] == i) | (i[:, None] == i)).float()  # itself and its parent
    for _ in range(max(1, (T - 1).bit_length())):
        a = (a @ a > 0).float()
    r = torch.arange(cols, device="cuda")
    j = r - s["rows"][:, None]
    tree = a.bool().gather(2, j.clamp(0, T - 1)[:, None].expand(-1, T, -1))
    return (j < 0)[:, None] | (tree & ((j >= 0) & (j < s["n_tok"][:, None]))[:, None])


def _plain_tree(s):
    c, B, T, Hkv, D = s["c"], s["B"], s["T"], s["Hkv"], s["D"]
    G = s["H"] // Hkv
    pages = s["table"].clamp(min=0).long()
    k = _load(s["K"][pages].flatten(1, 2), c["kv"], torch.float32).transpose(1, 2)  # [B, Hkv, rows, D]
    v = _load(s["V"][pages].flatten(1, 2), c["kv"], torch.float32).transpose(1, 2)
    seen = _seen(s, k.shape[2])
    q = s["q"].float().unflatten(2, (Hkv, G)).permute(0, 2, 3, 1, 4).reshape(B, Hkv, G * T, D)
    x = (q @ k.transpose(2, 3)).mul_(1.0 / math.sqrt(D)).unflatten(2, (G, T))
    x.masked_fill_(~seen[:, None, None], -math.inf)
    m = x.amax(-1, keepdim=True).clamp(min=-3e38)
    x = x.sub_(m).exp_()
    z = x.sum(-1, keepdim=True)
    o = (x.flatten(2, 3) @ v).unflatten(2, (G, T)) / z
    live = torch.arange(T, device="cuda") < s["n_tok"][:, None]
    o = o.permute(0, 3, 1, 2, 4).flatten(2, 3)
    s["out"].copy_(torch.where(live[..., None, None], o.to(s["out"].dtype), s["out"]))
    if s["lse"] is not None:
        lse = (m + z.log())[..., 0].permute(0, 3, 1, 2).flatten(2, 3)
        s["lse"].copy_(torch.where(live[..., None], lse, s["lse"]))


def _plain_pages(s):
    c, pools, P = s["c"], s["pools"], s["c"]["page"]
    if c["part"] == "copy":
        pools[:, s["to"].long()] = pools[:, s["from"].long()]
        return
    if c["part"] == "compact":
        j = torch.arange(s["path"].shape[1], device="cuda")
        live = j < s["n_path"][:, None]
        at = lambda r: (s["table"].gather(1, r // P).long() * P + r % P)[live]  # noqa: E731
        src = at(s["rows"][:, None].long() + s["path"])
        dst = at(s["rows"][:, None].long() + j)
        flat = pools.flatten(1, 2)
        flat[:, dst] = flat[:, src]
        s["rows_out"].copy_(s["rows"] + s["n_path"])
        return
    table, rows, refs = s["table"], s["rows"], s["refs"]
    to, frm = s["to"].long(), s["from"].long()
    held = table[to]
    refs.index_add_(0, held[held >= 0].long(), torch.full_like(held[held >= 0], -1))
    table[to], rows[to] = -1, 0
    full, part = rows[frm] // P, rows[frm] % P
    takes = (part > 0).int()
    rank = (takes.cumsum(0) - takes).long()
    free = torch.argsort((refs != 0).int(), stable=True)[rank].int()
    ok = (takes == 0) | (rank < (refs == 0).sum())
    col = torch.arange(table.shape[1], device="cuda")
    shared = (col < full[:, None]) & ok[:, None]
    mine = (col == full[:, None]) & (takes > 0)[:, None] & ok[:, None]
    old = table[frm]
    table[to] = torch.where(shared, old, torch.where(mine, free[:, None], torch.full_like(old, -1)))
    rows[to] = torch.where(ok, rows[frm], torch.zeros_like(part))
    refs.index_add_(0, old[shared].long(), torch.ones_like(old[shared]))
    copied = (takes > 0) & ok
    refs[free[copied].long()] = 1
    s["done"].copy_(ok.int())
    src = old.gather(1, full[:, None].clamp(max=table.shape[1] - 1).long())[copied].long()
    live = (torch.arange(P, device="cuda") < part[copied][:, None])[None, :, :, None, None]
    dst = free[copied].long()
    pools[:, dst] = torch.where(live, pools[:, src[:, 0]], pools[:, dst])


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------

def exact(case, seed):
    if case["op"] == "pages":
        return None  # moves and counts: whole numbers
    s = prepare(case, seed)
    return _exact_rope(s) if case["op"] == "rope" else _exact_tree(s)


def _exact_rope(s):
    c, D, n = s["c"], s["D"], s["c"]["n_rot"]
    P, Hkv = c["page"], s["Hkv"]
    d = torch.arange(D, device="cuda")
    # element d turns with its partner by the angle of rotary index i, with a sign of its own
    if c["mode"] == "halves":
        i, partner, sign = d % (n // 2), torch.where(d < n // 2, d + n // 2, d - n // 2), torch.where(d < n // 2, -1.0, 1.0)
    else:
        i, partner, sign = d // 2, d ^ 1, torch.where(d % 2 == 0, -1.0, 1.0)
    turned = d < n
    partner = torch.where(turned, partner, d)
    rate = torch.exp(i.double() * (-2.0 / n) * math.log(1e7)) * turned
    out = s["out"].double()
    k, v = (torch.zeros((t.shape[0] * P, Hkv, D), dtype=torch.float64, device="cuda") for t in (s["K"], s["V"]))
    held, new, table = s["rows"].tolist(), s["n_tok"].tolist(), s["table"].tolist()
    for b in range(s["B"]):
        t = new[b]
        a = s["pos"][b, :t].double()[:, None, None] * rate

        def turn(x, w):
            x = x.double()
            x = x / ((x * x).sum(-1, keepdim=True) / D + 1e-6).sqrt() * w.double()
            return x * a.cos() + (x[..., partner] * sign.double()) * a.sin() * turned

        out[b, :t] = turn(s["q"][b, :t], s["wq"])
        at = torch.tensor([table[b][r // P] * P + r % P for r in range(held[b], held[b] + t)], device="cuda")
        k[at], v[at] = turn(s["k"][b, :t], s["wk"]), s["v"][b, :t].double()
    if c["kv"] == "e5m2":  # its two bits of mantissa belong to what is stored: half first, then e5m2
        k, v = (x.half().to(torch.float8_e5m2).double() for x in (k, v))
    return {"q": out, "k": k, "v": v}


def _exact_tree(s):
    c, Hkv, D, P = s["c"], s["Hkv"], s["D"], s["c"]["page"]
    G = s["H"] // Hkv
    if sum(r * t for r, t in zip(s["rows"].tolist(), s["n_tok"].tolist())) * s["H"] * D > 6e11:
        return None
    out = s["out"].double()
    lse = None if s["lse"] is None else s["lse"].double()
    for b, (r, t) in enumerate(zip(s["rows"].tolist(), s["n_tok"].tolist())):
        n = r + t
        pages = s["table"][b, :_cdiv(n, P)].long()
        up = s["parents"][b].tolist()
        seen = torch.zeros((t, n), dtype=torch.bool)
        seen[:, :r] = True
        for i in range(t):
            j = i
            while j >= 0:
                seen[i, r + j] = True
                j = up[j]
        seen = seen.cuda()
        for h in range(Hkv):
            k, v = (_load(p[pages, :, h].flatten(0, 1)[:n], c["kv"], torch.float64) for p in (s["K"], s["V"]))
            for e in range(G):
                x = s["q"][b, :t, h * G + e].double() @ k.T / math.sqrt(D)
                x = torch.where(seen, x, -math.inf)
                z = torch.logsumexp(x, -1)
                out[b, :t, h * G + e] = torch.exp(x - z[:, None]) @ v
                if lse is not None:
                    lse[b, :t, h * G + e] = z
    return {"out": out, "lse": lse}
