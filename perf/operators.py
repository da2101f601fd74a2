"""Cases of the operators that serve many requests over shared Libraries.

read_shared   the routed read with every page fetched once for all rows that read it
pages_fork    child page tables that share a parent's pages, with fresh copies of the chunks the child owns
pages_compact live pages moved to the front of every pool, page tables renamed
adapt_in/out  the interface projections with a low-rank adapter per request beside the shared weight
"""

import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
READ_TEMP, ROUTE_TEMP, EPS = 12.0, 10.0, 1e-6


def listed():
    return [
        # a few tokens on one small document: launch latency
        dict(name="shared_small", op="read_shared", n_lib=1, rows=4, shared=8, private=0, page_rows=96, d_s=256, top_k=2,
             slots="f16", out="f32", softmax=True),
        # one decode step of 64 requests that ask about the same document of 64 chunks, top-4 routing
        dict(name="shared_decode", op="read_shared", n_lib=1, rows=64, shared=64, private=0, page_rows=512, d_s=2048,
             top_k=4, slots="f16", out="f32", softmax=True),
        # one decode step of 32 forks of a document (48 chunks in common, 16 of their own), dense routing
        dict(name="shared_prefix", op="read_shared", n_lib=32, rows=1, shared=48, private=16, page_rows=512, d_s=2048,
             top_k=0, slots="f16", out="f32", softmax=True),
        # two prompts of 2048 tokens over the same document, top-4 routing, bfloat16 hidden states
        dict(name="shared_prompt", op="read_shared", n_lib=2, rows=2048, shared=64, private=0, page_rows=512, d_s=2048,
             top_k=4, slots="f16", out="bf16", softmax=True),
        # a fork of a small Library at two depths: launch latency
        dict(name="fork_small", op="pages_fork", layers=2, n_lib=4, chunks=6, children=4, private=1, page_rows=64,
             d_s=256, slots="f16"),
        # 32 requests admitted at once, each with its own copy of the last two chunks, four depths
        dict(name="fork_batch", op="pages_fork", layers=4, n_lib=8, chunks=16, children=32, private=2, page_rows=512,
             d_s=2048, slots="f16"),
        # a small pool after a few requests left
        dict(name="compact_small", op="pages_compact", layers=2, n_lib=4, chunks=6, pages=64, page_rows=64, d_s=256,
             slots="f16"),
        # a pool half of whose pages were freed, four depths
        dict(name="compact_pool", op="pages_compact", layers=4, n_lib=8, chunks=16, pages=256, page_rows=512, d_s=2048,
             slots="f16"),
        # one token with its adapter
        dict(name="adapt_in_one", op="adapt_in", rows=1, rows_per_adapter=1, n_adapters=4, rank=8, d_in=4096,
             d_out=2048, h="bf16", adapters="bf16"),
        # a decode step of 64 requests, each with its own adapter
        dict(name="adapt_in_decode", op="adapt_in", rows=64, rows_per_adapter=1, n_adapters=64, rank=16, d_in=4096,
             d_out=2048, h="bf16", adapters="bf16"),
        # the same step's projection back into the reader
        dict(name="adapt_out_decode", op="adapt_out", rows=64, rows_per_adapter=1, n_adapters=64, rank=16, d_in=2048,
             d_out=4096, h="bf16", adapters="bf16"),
        # four prompts of 512 tokens, each with its own adapter
        dict(name="adapt_in_prompt", op="adapt_in", rows=2048, rows_per_adapter=512, n_adapters=4, rank=32, d_in=5120,
             d_out=2048, h="bf16", adapters="bf16"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["read_shared", "read_shared", "pages_fork", "pages_compact", "adapt_in", "adapt_out"])
    if op == "read_shared":
        prompt = rng.random() < 0.35
        n_lib = _log_int(rng, 1, 4) if prompt else _log_int(rng, 1, 32)
        rows = _log_int(rng, 128, 1024) if prompt else _log_int(rng, 1, max(1, 64 // n_lib))
        shared = _log_int(rng, 2, 48)
        private = 0 if n_lib == 1 else rng.randint(0, max(1, 96 // n_lib))
        top_k = rng.choice([0, 1, 2, 3, 4, 5, 8])
        if prompt:
            top_k = rng.choice([1, 2, 3, 4])
        return dict(op=op, n_lib=n_lib, rows=rows, shared=shared, private=private, page_rows=_log_int(rng, 17, 700),
                    d_s=8 * _log_int(rng, 8, 320), top_k=top_k, slots="f16" if not prompt else rng.choice(["f16", "bf16"]),
                    out="bf16" if prompt else rng.choice(["f32", "f32", "bf16"]), softmax=rng.random() < 0.8)
    if op in ("pages_fork", "pages_compact"):
        case = dict(op=op, layers=rng.randint(1, 5), n_lib=_log_int(rng, 1, 12), chunks=rng.randint(2, 16),
                    page_rows=_log_int(rng, 16, 512), d_s=8 * _log_int(rng, 8, 256), slots=rng.choice(["f16", "bf16"]))
        if op == "pages_fork":
            case.update(children=_log_int(rng, 1, 32), private=rng.randint(1, 2))
        else:
            case.update(pages=case["n_lib"] * case["chunks"] * 2 + rng.randint(1, 60))
        return case
    rpa = rng.choice([1, 1, _log_int(rng, 2, 500)])
    rows = rpa * _log_int(rng, 1, max(1, min(100, 2048 // rpa)))
    return dict(op=op, rows=rows, rows_per_adapter=rpa, n_adapters=_log_int(rng, 1, 80), rank=_log_int(rng, 2, 64),
                d_in=8 * _log_int(rng, 32, 512), d_out=8 * _log_int(rng, 32, 512), h=rng.choice(["bf16", "f16", "f32"]),
                adapters=rng.choice(["bf16", "f16"]))


# ------------------------------------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _unit(x):
    return x / x.norm(dim=-1, keepdim=True)


def _library_tables(case, g):
    """Page table and valid-row counts of n_lib Libraries whose first `shared` chunks are the same pages."""
    n_lib, sh, pv, N = case["n_lib"], case["shared"], case["private"], case["page_rows"]
    n_pages = sh + n_lib * pv
    order = torch.randperm(n_pages, generator=g, device="cuda")
    common = torch.arange(sh, device="cuda").expand(n_lib, sh)
    mine = sh + torch.arange(n_lib * pv, device="cuda").view(n_lib, pv)
    page_of = order[torch.cat([common, mine], 1)].to(torch.int32).contiguous()
    # chunks are full but for the last of the common part and the last of each Library's own part
    n_valid = torch.full((n_lib, sh + pv), N, dtype=torch.int32, device="cuda")
    n_valid[:, sh - 1] = int(torch.randint(1, N + 1, (1,), generator=g, device="cuda"))
    if pv:
        n_valid[:, -1] = torch.randint(1, N + 1, (n_lib,), generator=g, device="cuda", dtype=torch.int32)
    rows_of = torch.zeros(n_pages, dtype=torch.int64, device="cuda")
    rows_of[page_of.reshape(-1).long()] = n_valid.reshape(-1).long()
    return n_pages, page_of, n_valid, rows_of


def _prepare_read(case, seed):
    g = _gen(seed)
    n_lib, T, N, d = case["n_lib"], case["rows"], case["page_rows"], case["d_s"]
    n_pages, page_of, n_valid, rows_of = _library_tables(case, g)
    slots = _unit(torch.randn(n_pages, N, d, generator=g, device="cuda")).to(DTYPES[case["slots"]])
    slots *= (torch.arange(N, device="cuda") < rows_of[:, None])[..., None].to(slots.dtype)
    C = page_of.shape[1]
    # each query leans towards one slot of its Library, as a trained interface does
    lib = torch.arange(n_lib, device="cuda").repeat_interleave(T)
    near = torch.randint(0, C, (n_lib * T,), generator=g, device="cuda")
    at = (torch.rand(n_lib * T, generator=g, device="cuda") * n_valid[lib, near]).long()
    lean = torch.rand(n_lib * T, 1, generator=g, device="cuda") * 0.7
    q = _unit(_unit(torch.randn(n_lib * T, d, generator=g, device="cuda")) + lean * slots[page_of[lib, near].long(), at].float())
    mean = torch.stack([slots[p].float().sum(0) for p in range(n_pages)])
    S = _unit(mean)[page_of.long()]
    logits = torch.bmm(q.view(n_lib, T, d), S.transpose(1, 2)).reshape(n_lib * T, C) * ROUTE_TEMP
    k = case["top_k"] if 0 < case["top_k"] < C else C
    top, idx = logits.topk(k, dim=-1)
    wk = torch.softmax(top, -1)
    if n_lib * T > 8:  # a token that a LayerSelector drops reads nothing
        wk[5] = 0.0
    return dict(case=case, q=q, slots=slots, page_of=page_of, n_valid=n_valid, S=S.contiguous(),
                idx=idx.to(torch.int32).contiguous(), wk=wk.contiguous())


def _prepare_pages(case, seed):
    g = _gen(seed)
    n_lib, C, N, d = case["n_lib"], case["chunks"], case["page_rows"], case["d_s"]
    m, pv = case.get("children", 0), case.get("private", 0)
    n_pages = case["pages"] if "pages" in case else n_lib * C + m * pv + 16
    order = torch.randperm(n_pages, generator=g, device="cuda")
    page_of = order[: n_lib * C].view(n_lib, C).to(torch.int32).contiguous()
    page_of[:, 0] = page_of[0, 0]  # the Libraries were forked from one another: they begin with the same chunk
    n_valid = torch.full((n_lib, C), N, dtype=torch.int32, device="cuda")
    n_valid[:, -1] = torch.randint(1, N + 1, (n_lib,), generator=g, device="cuda", dtype=torch.int32)
    pools = [torch.randn(n_pages, N, d, generator=g, device="cuda").to(DTYPES[case["slots"]])
             for _ in range(case["layers"])]
    state = dict(case=case, pools=pools, page_of=page_of, n_valid=n_valid)
    if m:
        state["parents"] = torch.randint(0, n_lib, (m,), generator=g, device="cuda", dtype=torch.int32)
        state["own_from"] = torch.full((m,), C - pv, dtype=torch.int32, device="cuda")
    return state


def _prepare_adapters(case, seed):
    g = _gen(seed)
    R, d_in, d_out, r, n = case["rows"], case["d_in"], case["d_out"], case["rank"], case["n_adapters"]
    ad = DTYPES[case["adapters"]]
    n_of = R // case["rows_per_adapter"]
    of = torch.randperm(max(n, n_of), generator=g, device="cuda")[:n_of] % n
    if n_of > 8:
        of[3] = -1  # a request without an adapter
    x = torch.randn(R, d_in, generator=g, device="cuda")
    state = dict(case=case, of=of.to(torch.int32).contiguous(),
                 w=torch.randn(d_out, d_in, generator=g, device="cuda") * d_in ** -0.5,
                 a=(torch.randn(n, r, d_in, generator=g, device="cuda") * d_in ** -0.5).to(ad),
                 b=(torch.randn(n, d_out, r, generator=g, device="cuda") * 0.1).to(ad),
                 scale=torch.rand(n, generator=g, device="cuda") * 2 + 0.5)
    if case["op"] == "adapt_in":
        state["h"] = x.to(DTYPES[case["h"]])
    else:
        state["r"] = _unit(x)
        state["h"] = torch.randn(R, d_out, generator=g, device="cuda").to(DTYPES[case["h"]])
        state["gate"] = torch.rand(R, generator=g, device="cuda")
    if own:  # the weight in the form that the projections keep (once per interface)
        from kv_skill_v2_b200 import ops

        state["prep"] = ops.weights_prep(state["w"])
    return state


def prepare(case, seed):
    if case["op"] == "read_shared":
        return _prepare_read(case, seed)
    if case["op"] in ("pages_fork", "pages_compact"):
        return _prepare_pages(case, seed)
    return _prepare_adapters(case, seed)


# ------------------------------------------------------------------------------------------------- plain forms
def _plain_read(s):
    case = s["case"]
    n_lib, C = s["page_of"].shape
    R, d = s["q"].shape
    N = case["page_rows"]
    w = torch.zeros(R, C, device="cuda").scatter_add_(1, s["idx"].long(), s["wk"])
    K = s["slots"][s["page_of"].long()].float().view(n_lib, C * N, d)
    score = torch.bmm(s["q"].view(n_lib, -1, d), K.transpose(1, 2)).view(n_lib, -1, C, N)
    live = (torch.arange(N, device="cuda") < s["n_valid"][..., None])[:, None]
    if case["softmax"]:
        score = torch.where(live, score * READ_TEMP, float("-inf"))
        a = torch.exp(score - score.amax(-1, keepdim=True))
        a = a / a.sum(-1, keepdim=True)
    else:
        a = torch.where(live, score, 0.0) / s["n_valid"].float().sqrt()[:, None, :, None]
    aw = a * w.view(n_lib, -1, C, 1)
    return torch.bmm(aw.view(n_lib, -1, C * N), K).view(R, d).to(DTYPES[case["out"]])


def _copy_plain(pools, src, dst, rows):
    """Pages src -> dst of every pool: the first `rows` rows, zeros behind them."""
    keep = (torch.arange(pools[0].shape[1], device="cuda") < rows[:, None])[..., None]
    for p in pools:
        p[dst] = torch.where(keep, p[src], torch.zeros((), dtype=p.dtype, device="cuda"))


def _plain_fork(s):
    page_of, n_valid, parents = s["page_of"].long(), s["n_valid"], s["parents"].long()
    n_pages, C = s["pools"][0].shape[0], page_of.shape[1]
    used = torch.zeros(n_pages, dtype=torch.bool, device="cuda")
    used[page_of.reshape(-1)] = True
    free = torch.argsort(used.to(torch.int32), stable=True)  # free pages first, ascending
    child = page_of[parents]
    mine = torch.arange(C, device="cuda") >= s["own_from"][:, None]
    src = child[mine]
    dst = free[: src.numel()]
    _copy_plain(s["pools"], src, dst, n_valid[parents][mine])
    child = child.masked_scatter(mine, dst)
    short = torch.clamp(mine.sum() - (~used).sum(), min=0).to(torch.int32).view(1)
    return [child.to(torch.int32), short] + s["pools"]


def _plain_compact(s):
    page_of = s["page_of"].long()
    n_pages = s["pools"][0].shape[0]
    flat = page_of.reshape(-1)
    rows = torch.zeros(n_pages, dtype=torch.int32, device="cuda")
    rows = rows.scatter_reduce(0, flat, s["n_valid"].reshape(-1), "amax")
    used = torch.zeros(n_pages, dtype=torch.bool, device="cuda")
    used[flat] = True
    n_live = used.sum()
    low = torch.arange(n_pages, device="cuda") < n_live
    src = torch.nonzero(used & ~low).view(-1)
    dst = torch.nonzero(~used & low).view(-1)
    _copy_plain(s["pools"], src, dst, rows[src])
    to = torch.arange(n_pages, device="cuda")
    to[src] = dst
    return [to[page_of].to(torch.int32), n_live.to(torch.int32).view(1)] + s["pools"]


def _plain_adapt(s):
    case = s["case"]
    x = (s["h"] if case["op"] == "adapt_in" else s["r"]).float()
    R, d_in = x.shape
    of = s["of"].long()
    a, b = s["a"].float()[of.clamp(min=0)], s["b"].float()[of.clamp(min=0)]
    c = torch.where(of >= 0, s["scale"][of.clamp(min=0)], 0.0)
    if case["op"] == "adapt_in":
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    xg = x.view(of.numel(), -1, d_in)
    low = torch.bmm(torch.bmm(xg, a.transpose(1, 2)), b.transpose(1, 2)) * c[:, None, None]
    y = x @ s["w"].t() + low.reshape(R, -1)
    if case["op"] == "adapt_in":
        return y / (torch.sqrt((y * y).sum(-1, keepdim=True)) + EPS)
    return (y * s["gate"][:, None]).to(s["h"].dtype)


# ----------------------------------------------------------------------------------------------------------- run
def _own(s):
    from kv_skill_v2_b200 import ops

    case = s["case"]
    if case["op"] == "read_shared":
        pages = ops.Pages(slots=s["slots"], page_of=s["page_of"], n_valid=s["n_valid"], S=s["S"])
        return ops.read_shared(s["q"], pages, s["idx"], s["wk"], rows_per_lib=case["rows"], read_temp=READ_TEMP,
                               read_softmax=case["softmax"], out_dtype=DTYPES[case["out"]])
    if case["op"] == "pages_fork":
        return list(ops.pages_fork(s["pools"], s["page_of"], s["n_valid"], s["parents"], s["own_from"])) + s["pools"]
    if case["op"] == "pages_compact":
        return list(ops.pages_compact(s["pools"], s["page_of"], s["n_valid"])) + s["pools"]
    adapters = ops.Adapters(a=s["a"], b=s["b"], scale=s["scale"])
    more = dict(w_prep=s["prep"], adapters=adapters, adapter_of=s["of"], rows_per_adapter=case["rows_per_adapter"])
    if case["op"] == "adapt_in":
        return ops.project_in(s["h"], s["w"], **more)[0]
    return ops.project_out(s["r"], s["w"], s["h"], gate=s["gate"], **more)[0]


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    return {"read_shared": _plain_read, "pages_fork": _plain_fork, "pages_compact": _plain_compact,
            "adapt_in": _plain_adapt, "adapt_out": _plain_adapt}[op](state)


# ---------------------------------------------------------------------------------------------------------- work
def work(case):
    size = {"f32": 4, "f16": 2, "bf16": 2}
    if case["op"] == "read_shared":
        n_lib, T, d, N = case["n_lib"], case["rows"], case["d_s"], case["page_rows"]
        C, R = case["shared"] + case["private"], case["n_lib"] * case["rows"]
        k = case["top_k"] if 0 < case["top_k"] < C else C
        # pages that some row reads, each once
        pages = case["shared"] * (1 - (1 - k / C) ** R) + n_lib * case["private"] * (1 - (1 - k / C) ** T)
        return {"bytes": pages * N * d * size[case["slots"]] + R * d * (4 + size[case["out"]]) + R * k * 8,
                "flops": 4.0 * R * k * N * d}
    if case["op"] == "pages_fork":
        page = case["page_rows"] * case["d_s"] * size[case["slots"]]
        n = case["children"] * case["private"] * case["layers"]
        # the last of a child's own chunks is half full on average
        return {"bytes": n * page * 2.0 - case["children"] * case["layers"] * page * 0.5, "flops": 0.0}
    if case["op"] == "pages_compact":
        page = case["page_rows"] * case["d_s"] * size[case["slots"]]
        live = case["n_lib"] * (case["chunks"] - 1) + 1
        moved = live * (1 - live / case["pages"]) * case["layers"]
        return {"bytes": moved * page * (2.0 - 0.5 / case["chunks"]), "flops": 0.0}
    R, d_in, d_out, r = case["rows"], case["d_in"], case["d_out"], case["rank"]
    used = min(case["n_adapters"], R // case["rows_per_adapter"])
    x = size[case["h"]] * d_in + 4 * d_out if case["op"] == "adapt_in" else 4 * d_in + size[case["h"]] * d_out
    return {"bytes": 4.0 * d_in * d_out + used * r * (d_in + d_out) * size[case["adapters"]] + R * x,
            "flops": 2.0 * R * (d_in * d_out + r * (d_in + d_out))}


# --------------------------------------------------------------------------------------------- in 64 bits
def _exact_read(s):
    case = s["case"]
    q, T = s["q"].double(), case["rows"]
    out = torch.zeros_like(q)
    for lib in range(case["n_lib"]):
        mine = slice(lib * T, (lib + 1) * T)
        idx, wk = s["idx"][mine].long(), s["wk"][mine].double()
        for c in range(s["page_of"].shape[1]):
            weight = (wk * (idx == c)).sum(1)
            reads = weight.nonzero().view(-1)
            if reads.numel() == 0:
                continue
            n = int(s["n_valid"][lib, c])
            page = s["slots"][int(s["page_of"][lib, c]), :n].double()
            a = q[mine][reads] @ page.t()
            a = torch.softmax(READ_TEMP * a, -1) if case["softmax"] else a / math.sqrt(n)
            out[mine].index_add_(0, reads, weight[reads, None] * (a @ page))
    return out


def _exact_pages(s):
    case = s["case"]
    table, valid = s["page_of"].tolist(), s["n_valid"].tolist()
    n_pages = s["pools"][0].shape[0]
    live = sorted({p for row in table for p in row})
    moves = []
    if case["op"] == "pages_fork":
        free = [p for p in range(n_pages) if p not in set(live)]
        child = []
        for i, parent in enumerate(s["parents"].tolist()):
            row = list(table[parent])
            for c in range(int(s["own_from"][i]), len(row)):
                moves.append((row[c], free[0], valid[parent][c]))
                row[c] = free.pop(0)
            child.append(row)
        first = [torch.tensor(child, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)]
    else:
        n = len(live)
        holes = [p for p in range(n) if p not in set(live)]
        to = {p: p for p in live}
        for p in live:
            if p >= n:
                to[p] = holes.pop(0)
                rows = max(v for row, vs in zip(table, valid) for x, v in zip(row, vs) if x == p)
                moves.append((p, to[p], rows))
        first = [torch.tensor([[to[p] for p in row] for row in table], dtype=torch.int32),
                 torch.tensor([n], dtype=torch.int32)]
    pools = []
    for pool in s["pools"]:
        new = pool.double()
        for src, dst, rows in moves:
            new[dst, :rows] = pool[src, :rows].double()
            new[dst, rows:] = 0.0
        pools.append(new)
    return first + pools


def _exact_adapt(s):
    case = s["case"]
    x = (s["h"] if case["op"] == "adapt_in" else s["r"]).double()
    if case["op"] == "adapt_in":
        x = x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + EPS)
    y = torch.einsum("rk,nk->rn", x, s["w"].double())
    step = case["rows_per_adapter"]
    for i, a in enumerate(s["of"].tolist()):
        if a >= 0:
            rows = slice(i * step, (i + 1) * step)
            t = torch.einsum("rk,jk->rj", x[rows], s["a"][a].double())
            y[rows] += s["scale"][a].double() * torch.einsum("rj,nj->rn", t, s["b"][a].double())
    if case["op"] == "adapt_in":
        return y / (y.norm(dim=-1, keepdim=True) + EPS)
    return y * s["gate"].double()[:, None]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "read_shared":
        return _exact_read(s)
    return _exact_pages(s) if case["op"] in ("pages_fork", "pages_compact") else _exact_adapt(s)
