"""The operators of a serving step over a paged cache, as cases that can be timed and compared.

Three operators: the rotation of a step's queries and keys with the append of its keys and values to
the pages (``append``), attention of every sequence's new tokens over its pages (``attend``), and the
draw of the next tokens from logits (``sample``).  ``listed`` names the sizes that matter by name,
``draw`` takes others from the same ranges, ``prepare`` builds what a program holds before the call,
``run`` makes the call (``own`` false: elementary torch operations; true: the framework's kernels),
``work`` counts what the call cannot do without and ``exact`` states the operator in 64 bits.
"""

from __future__ import annotations

import math
import random
import sys
from pathlib import Path

import numpy as np
import torch

own = False   # whether `run` calls the framework's kernels or the plain forms

DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}
MAX_ROWS = 64 * 4352   # cache rows of one KV head over all sequences, largest attention case
MAX_TOKENS = 2048      # new tokens of a step over all sequences
VOCAB = 151936


def listed() -> list[dict]:
    return [
        # one user in the middle of a chat: the smallest step there is, all latency
        _attend("attend_b1_613", [(1, 613)], 16),
        # one user, a long document behind the question
        _attend("attend_b1_20001", [(1, 20001)], 64),
        # the throughput case: 64 sequences, each with a history of its own
        _attend("attend_b64_ragged", _ragged(64, 1, 1, 512, 4352, 7), 16),
        # drafted tokens of 19 sequences are checked at once: four each, heads of 64, fp16
        _attend("attend_verify_b19", _ragged(19, 4, 4, 300, 1111, 8), 32, heads=(16, 8), dim=64, dtype="float16"),
        # a piece of a long prompt that is brought in 512 tokens at a time
        _attend("attend_chunk512_4608", [(512, 4608)], 16),
        # a whole prompt at once
        _attend("attend_prompt2048", [(2048, 2048)], 64),
        # a step as a server makes it: 30 sequences decode, two prompts of odd lengths come in; keys of the last 1024 positions
        _attend("attend_mixed_window", _ragged(30, 1, 1, 200, 4352, 9) + [(777, 777), (131, 2000)], 48, window=1024),
        # a decode step of the throughput case: 64 new rows
        _append("append_t64", 64, 16),
        # a prompt of 2048 tokens, queries, keys and values as columns of one projection
        _append("append_t2048", 2048, 64, dtype="float16", tables="float32"),
        # one user with the usual settings
        _sample("sample_b1", 1, VOCAB, "bfloat16", "all"),
        # the throughput case, each sequence with settings of its own
        _sample("sample_b64", 64, VOCAB, "bfloat16", "mixed"),
        # no filter, logits in 32 bits: a token anywhere in the vocabulary
        _sample("sample_b8_open", 8, VOCAB, "float32", "open"),
    ]


def _ragged(batch: int, lo_q: int, hi_q: int, lo: int, hi: int, seed: int) -> list[tuple[int, int]]:
    """(new tokens, keys behind and with them) of each sequence, evenly over the logarithm of the history."""
    r = random.Random(seed)
    return [(r.randint(lo_q, hi_q), max(hi_q, round(lo * (hi / lo) ** r.random()))) for _ in range(batch)]


def _attend(name, seqs, page, heads=(12, 2), dim=128, dtype="bfloat16", window=0) -> dict:
    # the sequences as text: a case is a dict of plain values
    return {"name": name, "kind": "attend", "seqs": " ".join(f"{q}/{n}" for q, n in seqs), "page": page, "q_heads": heads[0],
            "kv_heads": heads[1], "dim": dim, "dtype": dtype, "window": window}


def _append(name, tokens, page, heads=(12, 2), dim=128, dtype="bfloat16", tables="") -> dict:
    return {"name": name, "kind": "append", "tokens": tokens, "page": page, "q_heads": heads[0], "kv_heads": heads[1], "dim": dim,
            "dtype": dtype, "tables": tables or dtype}


def _sample(name, rows, cols, dtype, filters) -> dict:
    return {"name": name, "kind": "sample", "rows": rows, "cols": cols, "dtype": dtype, "filters": filters}


def _seqs(case: dict) -> list[tuple[int, int]]:
    return [tuple(int(x) for x in s.split("/")) for s in case["seqs"].split()]


def _spread(rng, lo: int, hi: int) -> int:
    """A whole number from lo to hi, evenly over its logarithm."""
    return min(hi, max(lo, round(lo * (hi / lo) ** rng.random())))


def draw(rng) -> dict:
    kind = rng.choice(("attend", "attend", "attend", "append", "sample"))
    heads, dim = rng.choice((((12, 2), 128), ((12, 2), 128), ((16, 8), 64), ((8, 1), 128), ((6, 6), 128), ((14, 2), 64), ((32, 8), 128)))
    page, dtype = rng.choice((16, 16, 32, 48, 64, 128, 256)), rng.choice(("bfloat16", "bfloat16", "float16"))
    if kind == "sample":
        cols = _spread(rng, 100, VOCAB)
        case = _sample("", _spread(rng, 1, 64), cols, rng.choice(("bfloat16", "float16", "float32")), rng.choice(("all", "mixed", "open", "nucleus")))
    elif kind == "append":
        case = _append("", _spread(rng, 1, MAX_TOKENS), page, heads, dim, dtype, rng.choice((dtype, "float32")))
    else:
        budget = MAX_ROWS * 2 * 128 // (heads[1] * dim)
        what = rng.choice(("decode", "decode", "chunks", "mixed"))
        if what == "decode":
            batch, few = _spread(rng, 1, 64), rng.choice((1, 1, 1, 2, 3))
            longest = min(32768, budget // batch)
            seqs = [(few, max(few, _spread(rng, 1, longest))) for _ in range(batch)]
        else:
            # in work no more than the whole prompt of the largest listed case
            seqs, left = [], 4.0 * 128 * 12 * MAX_TOKENS * MAX_TOKENS / 2
            if what == "mixed":
                seqs = [(1, _spread(rng, 1, 4352)) for _ in range(_spread(rng, 1, 32))]
            for _ in range(rng.choice((1, 1, 2, 4))):
                q = _spread(rng, 2, 1024)
                n = q + rng.choice((0, _spread(rng, 1, 8192)))
                cost = 4.0 * dim * heads[0] * q * (n - q / 2)
                if cost <= left:
                    seqs.append((q, n))
                    left -= cost
            seqs = seqs or [(64, 300)]
            rng.shuffle(seqs)
        case = _attend("", seqs, page, heads, dim, dtype, rng.choice((0, 0, 0, 333, 1024)))
    del case["name"]
    return case


# ------------------------------------------------------------------ inputs
def _randn(shape, gen, dtype, scale=1.0):
    return (torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32) * scale).to(dtype)


def prepare(case: dict, seed: int) -> dict:
    gen = torch.Generator(device="cuda").manual_seed(seed)
    state = {"case": case, **{"attend": _prepare_attend, "append": _prepare_append, "sample": _prepare_sample}[case["kind"]](case, gen)}
    if own:
        path = str(Path.cwd() / "pytorch-apple_b200")
        if path not in sys.path:
            sys.path.insert(0, path)
        import paged_attention
        import sampling

        state["api"] = {"attend": paged_attention, "append": paged_attention, "sample": sampling}[case["kind"]]
    return state


def _prepare_attend(case: dict, gen) -> dict:
    seqs, page, dt = _seqs(case), case["page"], DTYPES[case["dtype"]]
    need = [-(-n // page) for _, n in seqs]
    n_pages = sum(need) + 3
    order = torch.randperm(n_pages, generator=gen, device="cuda").to(torch.int32)   # pages are handed out as they become free
    table = torch.zeros(len(seqs), max(need), dtype=torch.int32, device="cuda")
    at = 0
    for b, k in enumerate(need):
        table[b, :k] = order[at:at + k]
        at += k
    starts = np.concatenate([[0], np.cumsum([q for q, _ in seqs])])
    shape = (n_pages, case["kv_heads"], page, case["dim"])
    return {"q": _randn((int(starts[-1]), case["q_heads"], case["dim"]), gen, dt, 1.3), "k_pages": _randn(shape, gen, dt), "v_pages": _randn(shape, gen, dt),
            "q_start": torch.tensor(starts, dtype=torch.int32, device="cuda"),
            "kv_len": torch.tensor([n for _, n in seqs], dtype=torch.int32, device="cuda"), "table": table, "seqs": seqs,
            "max_q": max(q for q, _ in seqs), "scale": case["dim"] ** -0.5}


def _prepare_append(case: dict, gen) -> dict:
    N, page, dim, dt = case["tokens"], case["page"], case["dim"], DTYPES[case["dtype"]]
    hq, hkv = case["q_heads"], case["kv_heads"]
    qkv = _randn((N, (hq + 2 * hkv) * dim), gen, dt)   # one merged projection: the three are columns of its rows
    q, k, v = (t.unflatten(1, (-1, dim)) for t in qkv.split([hq * dim, hkv * dim, hkv * dim], 1))
    positions = torch.randint(0, 32768, (N,), generator=gen, device="cuda")
    angle = positions.double()[:, None] * (1e6 ** (-torch.arange(0, dim, 2, dtype=torch.float64, device="cuda") / dim))[None]
    angle = torch.cat([angle, angle], 1)
    n_pages = -(-2 * N // page) + 2
    slots = torch.randperm(n_pages * page, generator=gen, device="cuda")[:N].contiguous()
    shape = (n_pages, hkv, page, dim)
    return {"q": q, "k": k, "v": v, "cos": angle.cos().to(DTYPES[case["tables"]]), "sin": angle.sin().to(DTYPES[case["tables"]]), "slots": slots,
            "k_pages": _randn(shape, gen, dt), "v_pages": _randn(shape, gen, dt)}


def _prepare_sample(case: dict, gen) -> dict:
    rows, cols = case["rows"], case["cols"]
    # a wide bulk of tokens that hardly matter, and some hundred that do
    x = torch.randn(rows, cols, generator=gen, device="cuda") * 2.2
    liked = torch.rand(rows, cols, generator=gen, device="cuda") < 300.0 / cols
    x += liked * (4.0 - 3.0 * torch.rand(rows, cols, generator=gen, device="cuda").log())
    u = lambda lo, hi: lo + (hi - lo) * torch.rand(rows, generator=gen, device="cuda")
    on = lambda share, value, off: torch.where(torch.rand(rows, generator=gen, device="cuda") < share, value, torch.full_like(value, off))
    st = {"logits": x.to(DTYPES[case["dtype"]]), "uniform": torch.rand(rows, generator=gen, device="cuda"), "temperature": u(0.6, 1.3),
          "top_k": None, "top_p": None, "min_p": None}
    k = (20 * 25 ** torch.rand(rows, generator=gen, device="cuda")).to(torch.int32)
    if case["filters"] == "all":
        st.update(top_k=k, top_p=u(0.8, 0.98), min_p=u(0.01, 0.1))
    elif case["filters"] == "nucleus":
        st.update(top_p=u(0.5, 0.99))
    elif case["filters"] == "mixed":   # some rows greedy, each filter on for most rows
        st.update(temperature=on(0.9, st["temperature"], 0.0), top_k=on(0.6, k, 0), top_p=on(0.7, u(0.8, 0.98), 1.0), min_p=on(0.4, u(0.01, 0.1), 0.0))
    return st


# ------------------------------------------------------------------ one pass
def run(state: dict):
    kind = state["case"]["kind"]
    if own:
        api = state["api"]
        if kind == "attend":
            return api.paged_attention(state["q"], state["k_pages"], state["v_pages"], state["q_start"], state["kv_len"], state["table"], state["max_q"],
                                       scale=state["scale"], window=state["case"]["window"])
        if kind == "append":
            q = api.paged_append(state["q"], state["k"], state["v"], state["cos"], state["sin"], state["k_pages"], state["v_pages"], state["slots"])
            return q, state["k_pages"], state["v_pages"]
        return api.sample_rows(state["logits"], state["uniform"], temperature=state["temperature"], top_k=state["top_k"], top_p=state["top_p"],
                               min_p=state["min_p"])
    return {"attend": _plain_attend, "append": _plain_append, "sample": _plain_sample}[kind](state)


def _plain_attend(s: dict):
    case, dt = s["case"], s["q"].dtype
    out, at = torch.empty_like(s["q"]), 0
    group = case["q_heads"] // case["kv_heads"]
    for b, (T, n) in enumerate(s["seqs"]):
        ids = s["table"][b, :-(-n // case["page"])].long()
        k, v = (p[ids].transpose(0, 1).flatten(1, 2)[:, :n].float().repeat_interleave(group, 0) for p in (s["k_pages"], s["v_pages"]))
        scores = torch.matmul(s["q"][at:at + T].float().transpose(0, 1), k.transpose(1, 2)) * s["scale"]
        pos = torch.arange(n - T, n, device="cuda")[:, None]
        key = torch.arange(n, device="cuda")[None]
        unseen = key > pos
        if case["window"]:
            unseen = unseen | (key <= pos - case["window"])
        scores = scores.masked_fill(unseen, -math.inf)
        w = torch.exp(scores - scores.amax(-1, keepdim=True))
        out[at:at + T] = (torch.matmul(w, v) / w.sum(-1, keepdim=True)).transpose(0, 1).to(dt)
        at += T
    return out


def _plain_append(s: dict):
    page, half = s["case"]["page"], s["case"]["dim"] // 2
    cos, sin = s["cos"].float()[:, None], s["sin"].float()[:, None]

    def rotate(x):
        x = x.float()
        return x * cos + torch.cat([-x[..., half:], x[..., :half]], -1) * sin

    q = rotate(s["q"]).to(s["q"].dtype)
    where, row = s["slots"] // page, s["slots"] % page
    s["k_pages"][where, :, row] = rotate(s["k"]).to(s["k"].dtype)
    s["v_pages"][where, :, row] = s["v"]
    return q, s["k_pages"], s["v_pages"]


def _plain_sample(s: dict):
    x = s["logits"].double()   # sums over a vocabulary, and tokens next to a border: 64 bits
    rows, cols = x.shape
    greedy = s["temperature"] <= 0
    temp = torch.where(greedy, torch.ones_like(s["temperature"]), s["temperature"]).double()[:, None]
    top, order = torch.sort(x, dim=1, descending=True, stable=True)
    w = torch.exp((top - top[:, :1]) / temp)
    rank = torch.arange(cols, device="cuda")[None]
    keep = torch.ones_like(w, dtype=torch.bool)
    if s["top_k"] is not None:
        k = s["top_k"][:, None]
        keep = (rank < k) | (k <= 0)
    if s["top_p"] is not None:
        kept = w * keep
        before = kept.cumsum(1) - kept
        p = s["top_p"].double()[:, None]
        keep = keep & ((p >= 1) | (before < p * kept.sum(1, keepdim=True)) | (rank == 0))
    if s["min_p"] is not None:
        keep = keep & (w >= s["min_p"].double()[:, None].clamp(max=1.0))
    keep = keep & (~greedy[:, None] | (rank == 0))
    by_index = torch.zeros_like(w).scatter_(1, order, w * keep)
    total = by_index.cumsum(1)
    target = s["uniform"].double()[:, None] * total[:, -1:]
    return (total <= target).sum(1).clamp(max=cols - 1)


# ------------------------------------------------------------------ what a pass cannot do without
def _attended(T: int, n: int, window: int) -> tuple[int, int]:
    """(rows of the cache that some new token looks at, pairs of token and key)."""
    spans = [(max(0, p - window + 1) if window else 0, p + 1) for p in range(n - T, n)]
    return spans[-1][1] - spans[0][0], sum(hi - lo for lo, hi in spans)


def work(case: dict) -> dict:
    if case["kind"] == "sample":
        n = case["rows"] * case["cols"]
        size = 4 if case["dtype"] == "float32" else 2
        return {"bytes": n * size + case["rows"] * 28, "flops": 3 * n}   # difference, exponential, sum
    hq, hkv, dim = case["q_heads"], case["kv_heads"], case["dim"]
    if case["kind"] == "append":
        N, size = case["tokens"], 4 if case["tables"] == "float32" else 2
        return {"bytes": 2 * N * (hq + 2 * hkv) * dim * 2 + 2 * N * dim * size + 8 * N, "flops": 3 * N * (hq + hkv) * dim}
    rows = pairs = tokens = ids = 0
    for T, n in _seqs(case):
        r, p = _attended(T, n, case["window"])
        rows, pairs, tokens, ids = rows + r, pairs + p, tokens + T, ids + -(-r // case["page"])
    return {"bytes": rows * hkv * dim * 4 + tokens * hq * dim * 4 + 4 * ids, "flops": 4 * dim * hq * pairs}


# ------------------------------------------------------------------ the definition in 64 bits
def exact(case: dict, seed: int):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    return {"attend": _exact_attend, "append": _exact_append, "sample": _exact_sample}[case["kind"]](case, s)


def _exact_attend(case: dict, s: dict):
    hq, hkv, dim, page = case["q_heads"], case["kv_heads"], case["dim"], case["page"]
    q = s["q"].double().view(-1, hkv, hq // hkv, dim)
    # rows of the cache in a line: (page, row) of a KV head
    rows_k, rows_v = (p.permute(1, 0, 2, 3).reshape(hkv, -1, dim) for p in (s["k_pages"], s["v_pages"]))
    result, first = [], 0
    for b, (T, n) in enumerate(s["seqs"]):
        j = torch.arange(n, device="cuda")
        row = s["table"][b].long()[j // page] * page + j % page
        k, v = rows_k[:, row].double(), rows_v[:, row].double()
        for i0 in range(0, T, 64):   # some tokens at a time: the scores of all would be too many
            i = torch.arange(i0, min(T, i0 + 64), device="cuda")
            p = n - T + i
            score = torch.einsum("thgd,hjd->thgj", q[first + i], k) * s["scale"]
            seen = (j[None] <= p[:, None]) & ((j[None] > p[:, None] - case["window"]) if case["window"] else True)
            prob = torch.softmax(torch.where(seen[:, None, None], score, torch.full_like(score, -math.inf)), -1)
            result.append(torch.einsum("thgj,hjd->thgd", prob, v).reshape(-1, hq, dim))
        first += T
    return torch.cat(result)


def _exact_append(case: dict, s: dict):
    hkv, dim, page = case["kv_heads"], case["dim"], case["page"]
    c, si = (s[t].double().view(-1, 1, 2, dim // 2) for t in ("cos", "sin"))

    def turned(x):   # pairs (a, b) of the two halves: (a cos - b sin, b cos + a sin)
        a, b = x.double().unflatten(-1, (2, -1)).unbind(-2)
        return torch.stack([a * c[:, :, 0] - b * si[:, :, 0], b * c[:, :, 1] + a * si[:, :, 1]], -2).flatten(-2)

    pools = []
    for name, new in (("k_pages", turned(s["k"])), ("v_pages", s["v"].double())):
        flat = s[name].double().permute(0, 2, 1, 3).reshape(-1, hkv, dim)
        flat[s["slots"]] = new
        pools.append(flat.view(-1, page, hkv, dim).permute(0, 2, 1, 3).contiguous())
    return turned(s["q"]), pools[0], pools[1]


def _exact_sample(case: dict, s: dict):
    cpu = lambda t: None if t is None else t.double().cpu().numpy()
    x, u, temp, ks, ps, ms = (cpu(s[n]) for n in ("logits", "uniform", "temperature", "top_k", "top_p", "min_p"))
    tokens = []
    for r in range(case["rows"]):
        if temp[r] <= 0:
            tokens.append(int(np.argmax(x[r])))
            continue
        rank = np.argsort(-x[r], kind="stable")
        if ks is not None and ks[r] > 0:
            rank = rank[:int(ks[r])]
        w = np.exp((x[r][rank] - x[r].max()) / temp[r])
        if ps is not None and ps[r] < 1:
            sums = np.concatenate([[0.0], np.cumsum(w)])
            count = max(1, int(np.searchsorted(sums[:-1], ps[r] * sums[-1], side="left")))
            rank, w = rank[:count], w[:count]
        if ms is not None:
            alive = w >= min(ms[r], 1.0)
            rank, w = rank[alive], w[alive]
        by_index = np.argsort(rank)
        sums = np.cumsum(w[by_index])
        tokens.append(int(rank[by_index][min(len(sums) - 1, np.searchsorted(sums, u[r] * sums[-1], side="right"))]))
    return torch.tensor(tokens, device="cuda")
