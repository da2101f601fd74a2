"""Cases of the operators that shrink a served Library and put its interface into 8 bits.

read_mass    the attention that every slot of a pool receives from a batch of rows, added to what it had before
pages_evict  the slots with most of it stay, in their order, at the front of new (smaller) pages
in8, out8    the interface projections in 8-bit floating point, a power of two for each row's block of 128 columns
"""

import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
READ_TEMP, ROUTE_TEMP, EPS = 12.0, 10.0, 1e-6
BLOCK, E4M3_MAX = 128, 448.0


def listed():
    return [
        # a few tokens on one small document: launch latency
        dict(name="mass_small", op="read_mass", n_lib=1, rows=4, shared=8, private=0, page_rows=96, d_s=256, top_k=2,
             slots="f16", q="f32", decay=1.0),
        # one decode step of 64 requests on a document of 64 chunks, top-4 routing, older attention fading
        dict(name="mass_decode", op="read_mass", n_lib=1, rows=64, shared=64, private=0, page_rows=512, d_s=2048,
             top_k=4, slots="f16", q="f32", decay=0.95),
        # two prompts of 2048 tokens over the same document, top-4 routing: what the eviction after a prompt goes by
        dict(name="mass_prompt", op="read_mass", n_lib=2, rows=2048, shared=64, private=0, page_rows=512, d_s=2048,
             top_k=4, slots="f16", q="f32", decay=1.0),
        # a small Library at two depths, each chunk to a quarter of its slots: launch latency
        dict(name="evict_small", op="pages_evict", layers=2, n_lib=4, chunks=6, pages=40, page_rows=64, d_s=256,
             slots="f16", keep=16, new_rows=16, per_library=False, ragged=False),
        # one budget for a whole document, odd sizes, forks that read fewer rows of a shared page
        dict(name="evict_budget", op="pages_evict", layers=2, n_lib=5, chunks=37, pages=220, page_rows=203, d_s=1032,
             slots="bf16", keep=2501, new_rows=150, per_library=True, ragged=True),
        # eight documents of 16 chunks at four depths, each chunk from 512 to 128 slots
        dict(name="evict_pool", op="pages_evict", layers=4, n_lib=8, chunks=16, pages=128, page_rows=512, d_s=2048,
             slots="f16", keep=128, new_rows=128, per_library=False, ragged=False),
        # one token into the encoder's space
        dict(name="in8_one", op="in8", rows=1, d_in=4096, d_out=2048, h="bf16"),
        # a decode step of 64 requests
        dict(name="in8_decode", op="in8", rows=64, d_in=4096, d_out=2048, h="bf16"),
        # a prompt of 2048 tokens of a wider reader
        dict(name="in8_prompt", op="in8", rows=2048, d_in=5120, d_out=2048, h="bf16"),
        # a small interface of odd widths
        dict(name="out8_odd", op="out8", rows=5, d_in=328, d_out=1000, h="f32"),
        # a decode step back into the reader
        dict(name="out8_decode", op="out8", rows=64, d_in=2048, d_out=4096, h="bf16"),
        # eight prompts of 2048 tokens back into the reader
        dict(name="out8_prompts", op="out8", rows=16384, d_in=2048, d_out=4096, h="bf16"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["read_mass", "read_mass", "pages_evict", "pages_evict", "in8", "out8"])
    if op == "read_mass":
        prompt = rng.random() < 0.4
        n_lib = _log_int(rng, 1, 4) if prompt else _log_int(rng, 1, 24)
        rows = _log_int(rng, 128, 1024) if prompt else _log_int(rng, 1, max(1, 64 // n_lib))
        shared = _log_int(rng, 2, 48)
        private = 0 if n_lib == 1 else rng.randint(0, max(1, 72 // n_lib))
        return dict(op=op, n_lib=n_lib, rows=rows, shared=shared, private=private, page_rows=_log_int(rng, 17, 700),
                    d_s=8 * _log_int(rng, 8, 320), top_k=rng.choice([1, 2, 3, 4] if prompt else [0, 1, 2, 3, 5, 8]),
                    slots=rng.choice(["f16", "f16", "bf16"]), q=rng.choice(["f32", "bf16", "f16"]),
                    decay=rng.choice([1.0, 0.9, 0.5]))
    if op == "pages_evict":
        per_library = rng.random() < 0.5
        n_lib, chunks, page_rows = _log_int(rng, 1, 10), _log_int(rng, 2, 40), _log_int(rng, 9, 600)
        new_rows = _log_int(rng, 3, page_rows)
        return dict(op=op, layers=rng.randint(1, 4), n_lib=n_lib, chunks=chunks, page_rows=page_rows,
                    pages=n_lib * chunks + rng.randint(0, 40), d_s=8 * _log_int(rng, 8, 160),
                    slots=rng.choice(["f16", "bf16", "f32"]), new_rows=new_rows, per_library=per_library,
                    keep=_log_int(rng, 1, new_rows * chunks) if per_library else rng.randint(1, new_rows),
                    ragged=rng.random() < 0.5)
    return dict(op=op, rows=_log_int(rng, 1, 4096), d_in=8 * _log_int(rng, 16, 640), d_out=8 * _log_int(rng, 16, 512),
                h=rng.choice(["bf16", "f16", "f32"]))


# ------------------------------------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _unit(x):
    return x / x.norm(dim=-1, keepdim=True)


def _prepare_mass(case, seed):
    g = _gen(seed)
    n_lib, T, N, d = case["n_lib"], case["rows"], case["page_rows"], case["d_s"]
    sh, pv = case["shared"], case["private"]
    n_pages = sh + n_lib * pv
    # the Libraries' first chunks are the same pages, the rest their own; full but for the last of each part
    order = torch.randperm(n_pages, generator=g, device="cuda")
    common = torch.arange(sh, device="cuda").expand(n_lib, sh)
    mine = sh + torch.arange(n_lib * pv, device="cuda").view(n_lib, pv)
    page_of = order[torch.cat([common, mine], 1)].to(torch.int32).contiguous()
    n_valid = torch.full((n_lib, sh + pv), N, dtype=torch.int32, device="cuda")
    last = sh - 1 if pv == 0 else sh + pv - 1
    n_valid[:, last] = torch.randint(1, N + 1, (n_lib,), generator=g, device="cuda", dtype=torch.int32)
    slots = _unit(torch.randn(n_pages, N, d, generator=g, device="cuda")).to(DTYPES[case["slots"]])
    C = sh + pv
    # each query leans towards one slot of its Library, as a trained interface does
    lib = torch.arange(n_lib, device="cuda").repeat_interleave(T)
    near = torch.randint(0, C, (n_lib * T,), generator=g, device="cuda")
    at = (torch.rand(n_lib * T, generator=g, device="cuda") * n_valid[lib, near]).long()
    lean = torch.rand(n_lib * T, 1, generator=g, device="cuda") * 0.7
    q = _unit(_unit(torch.randn(n_lib * T, d, generator=g, device="cuda"))
              + lean * slots[page_of[lib, near].long(), at].float())
    S = _unit(torch.stack([slots[p].float().sum(0) for p in range(n_pages)]))[page_of.long()]
    logits = torch.bmm(q.view(n_lib, T, d), S.transpose(1, 2)).reshape(n_lib * T, C) * ROUTE_TEMP
    k = case["top_k"] if 0 < case["top_k"] < C else C
    top, idx = logits.topk(k, dim=-1)
    wk = torch.softmax(top, -1)
    if n_lib * T > 8:  # a token that a LayerSelector drops reads nothing
        wk[5] = 0.0
    # what earlier batches of this size left
    prior = torch.rand(n_pages, N, generator=g, device="cuda") * (2.0 * n_lib * T / (n_pages * N))
    return dict(case=case, q=q.to(DTYPES[case["q"]]), slots=slots, page_of=page_of, n_valid=n_valid, S=S.contiguous(),
                idx=idx.to(torch.int32).contiguous(), wk=wk.contiguous(), prior=prior)


def _prepare_evict(case, seed):
    g = _gen(seed)
    n_lib, C, N, d, P = case["n_lib"], case["chunks"], case["page_rows"], case["d_s"], case["pages"]
    order = torch.randperm(P, generator=g, device="cuda")
    page_of = order[: n_lib * C].view(n_lib, C).to(torch.int32).contiguous()
    page_of[:, 0] = page_of[0, 0]  # the Libraries were forked from one another: they begin with the same chunk
    n_valid = torch.full((n_lib, C), N, dtype=torch.int32, device="cuda")
    n_valid[:, -1] = torch.randint(1, N + 1, (n_lib,), generator=g, device="cuda", dtype=torch.int32)
    if case["ragged"]:
        n_valid[:] = torch.randint(max(1, N // 2), N + 1, (n_lib, C), generator=g, device="cuda", dtype=torch.int32)
    # attention is heavy-tailed; a fifth of the slots never got any
    mass = torch.exp(2.0 * torch.randn(P, N, generator=g, device="cuda"))
    mass = torch.where(torch.rand(P, N, generator=g, device="cuda") < 0.2, 0.0, mass)
    pools = [torch.randn(P, N, d, generator=g, device="cuda").to(DTYPES[case["slots"]]) for _ in range(case["layers"])]
    shape = (n_lib,) if case["per_library"] else (n_lib, C)
    keep = torch.full(shape, case["keep"], dtype=torch.int32, device="cuda")
    return dict(case=case, pools=pools, page_of=page_of, n_valid=n_valid, mass=mass, keep=keep)


def _blocks(x):
    """(values [n, 128 B] in e4m3, exponents [n, B] int32): x [n, k] in blocks of 128 columns (zeros behind the last), each
    times the smallest power of two 2^-e that brings it to at most 448."""
    n, k = x.shape
    x = torch.nn.functional.pad(x.float(), (0, -k % BLOCK)).view(n, -1, BLOCK)
    m, e = torch.frexp(x.abs().amax(-1))  # the largest is m 2^e, m in [1/2, 1); 448 = (7/8) 2^9
    e = torch.where(m == 0, 0, e - 9 + (m > E4M3_MAX / 512).to(torch.int32)).clamp(-127, 127)
    return torch.ldexp(x, -e[..., None]).to(torch.float8_e4m3fn).view(n, -1), e


def _prepare_project(case, seed):
    g = _gen(seed)
    R, d_in, d_out = case["rows"], case["d_in"], case["d_out"]
    # hidden states have a few channels that are much larger than the others
    loud = torch.exp(1.5 * torch.randn(d_in, generator=g, device="cuda"))
    x = torch.randn(R, d_in, generator=g, device="cuda") * loud
    w8, e = _blocks(torch.randn(d_out, d_in, generator=g, device="cuda") * d_in ** -0.5)
    state = dict(case=case, w8=w8, w_scale=(e + 127).to(torch.uint8).contiguous())
    if case["op"] == "in8":
        state["h"] = x.to(DTYPES[case["h"]])
        state["b"] = torch.randn(d_out, generator=g, device="cuda") * 0.1
    else:
        state["r"] = _unit(x)
        state["h"] = torch.randn(R, d_out, generator=g, device="cuda").to(DTYPES[case["h"]])
        state["gate"] = torch.rand(R, generator=g, device="cuda")
    return state


def prepare(case, seed):
    make = {"read_mass": _prepare_mass, "pages_evict": _prepare_evict, "in8": _prepare_project, "out8": _prepare_project}
    return make[case["op"]](case, seed)


# ------------------------------------------------------------------------------------------------- plain forms
def _plain_mass(s):
    case = s["case"]
    n_lib, C = s["page_of"].shape
    R, d = s["q"].shape
    N = case["page_rows"]
    w = torch.zeros(R, C, device="cuda").scatter_add_(1, s["idx"].long(), s["wk"])
    K = s["slots"][s["page_of"].long()].float().view(n_lib, C * N, d)
    score = torch.bmm(s["q"].float().view(n_lib, -1, d), K.transpose(1, 2)).view(n_lib, -1, C, N)
    live = (torch.arange(N, device="cuda") < s["n_valid"][..., None])[:, None]
    score = torch.where(live, score * READ_TEMP, float("-inf"))
    a = torch.exp(score - score.amax(-1, keepdim=True))
    a = a / a.sum(-1, keepdim=True)
    got = (a * w.view(n_lib, -1, C, 1)).sum(1)
    return (s["prior"] * case["decay"]).index_add_(0, s["page_of"].reshape(-1).long(), got.view(-1, N))


def _rank(x):
    """Each value's place in its row, the largest first, equal ones by their index."""
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices
    at = torch.arange(x.shape[-1], device="cuda").expand_as(order)
    return torch.empty_like(order).scatter_(-1, order, at)


def _plain_evict(s):
    case = s["case"]
    page_of, n_valid, keep = s["page_of"].long(), s["n_valid"].long(), s["keep"].long()
    (n_lib, C), (P, N), M = page_of.shape, s["mass"].shape, case["new_rows"]
    flat = page_of.reshape(-1)
    slot = torch.arange(N, device="cuda")
    rows = torch.zeros(P, dtype=torch.int64, device="cuda").scatter_reduce(0, flat, n_valid.reshape(-1), "amax")
    rank = _rank(torch.where(slot < rows[:, None], s["mass"], float("-inf")))  # among the rows that some table reads
    if case["per_library"]:
        first = (rank < 1) & (slot < rows[:, None])  # a page keeps its heaviest row
        may = (rank >= 1) & (rank < M) & (slot < rows[:, None])
        read = slot < n_valid[..., None]
        mine = (may[page_of] & read).view(n_lib, -1)
        left = keep - (first[page_of] & read).view(n_lib, -1).sum(-1)
        weight = torch.where(mine, s["mass"][page_of].view(n_lib, -1), float("-inf"))
        chosen = ((_rank(weight) < left[:, None]) & mine).view(-1, N)
        stays = torch.zeros(P, N, dtype=torch.int32, device="cuda").index_add_(0, flat, chosen.to(torch.int32)) > 0
        stays = stays | first
    else:
        most = torch.zeros(P, dtype=torch.int64, device="cuda").scatter_reduce(0, flat, keep.reshape(-1), "amax")
        stays = (rank < torch.minimum(most.clamp(min=1, max=M), rows)[:, None])
    left = (stays[page_of] & (slot < n_valid[..., None])).sum(-1)
    src = torch.sort((~stays).to(torch.int32), dim=-1, stable=True).indices[:, :M]  # the rows that stay, ascending
    there = torch.arange(M, device="cuda") < stays.sum(-1)[:, None]
    mass = torch.where(there, s["mass"].gather(1, src), 0.0)
    at = (torch.arange(P, device="cuda")[:, None] * N + src).view(-1)
    pools = [torch.where(there[..., None], p.view(P * N, -1)[at].view(P, M, -1), torch.zeros((), dtype=p.dtype, device="cuda"))
             for p in s["pools"]]
    return [left.to(torch.int32), mass, torch.where(there, src, -1).to(torch.int32)] + pools


def _plain_project(s):
    case = s["case"]
    R, d_in, d_out = case["rows"], case["d_in"], case["d_out"]
    x = (s["h"] if case["op"] == "in8" else s["r"]).float()
    x8, e = _blocks(x)
    xq = torch.ldexp(x8.float().view(R, -1, BLOCK), e[..., None]).view(R, -1)
    wq = torch.ldexp(s["w8"].float().view(d_out, -1, BLOCK), s["w_scale"].int()[..., None] - 127).view(d_out, -1)
    y = xq @ wq.t()
    if case["op"] == "out8":
        return (y * s["gate"][:, None]).to(s["h"].dtype)
    y = y * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) + s["b"]
    return y / (torch.sqrt((y * y).sum(-1, keepdim=True)) + EPS)


# ----------------------------------------------------------------------------------------------------------- run
def _own(s):
    from kv_skill_v2_b200 import ops

    case = s["case"]
    if case["op"] == "read_mass":
        pages = ops.Pages(slots=s["slots"], page_of=s["page_of"], n_valid=s["n_valid"], S=s["S"])
        return ops.read_mass(s["q"], pages, s["idx"], s["wk"], rows_per_lib=case["rows"], read_temp=READ_TEMP,
                             mass=s["prior"], decay=case["decay"])
    if case["op"] == "pages_evict":
        n_valid, mass, kept, pools = ops.pages_evict(s["pools"], s["page_of"], s["n_valid"], s["mass"], s["keep"],
                                                     per_library=case["per_library"], page_rows=case["new_rows"])
        return [n_valid, mass, kept] + pools
    w = ops.Weights8(w=s["w8"], scale=s["w_scale"], k=case["d_in"])
    if case["op"] == "in8":
        return ops.project_in(s["h"], w, s["b"])[0]
    return ops.project_out(s["r"], w, s["h"], gate=s["gate"])[0]


def run(state):
    if own:
        return _own(state)
    return {"read_mass": _plain_mass, "pages_evict": _plain_evict, "in8": _plain_project,
            "out8": _plain_project}[state["case"]["op"]](state)


# ---------------------------------------------------------------------------------------------------------- work
def work(case):
    size = {"f32": 4, "f16": 2, "bf16": 2}
    if case["op"] == "read_mass":
        n_lib, T, d, N = case["n_lib"], case["rows"], case["d_s"], case["page_rows"]
        C, R = case["shared"] + case["private"], case["n_lib"] * case["rows"]
        k = case["top_k"] if 0 < case["top_k"] < C else C
        # pages that some row reads, each once
        pages = case["shared"] * (1 - (1 - k / C) ** R) + n_lib * case["private"] * (1 - (1 - k / C) ** T)
        held = case["shared"] + n_lib * case["private"]
        return {"bytes": pages * N * d * size[case["slots"]] + R * d * size[case["q"]] + R * k * 8 + held * N * 8.0,
                "flops": 2.0 * R * k * N * d}
    if case["op"] == "pages_evict":
        live = case["n_lib"] * (case["chunks"] - 1) + 1
        N, M = case["page_rows"], case["new_rows"]
        if case["per_library"]:
            kept = min(live * M, case["n_lib"] * case["keep"])
        else:
            kept = live * min(case["keep"], M)
        row = case["d_s"] * size[case["slots"]] * case["layers"]
        return {"bytes": float(kept * row + case["pages"] * M * (row + 8) + live * N * 4), "flops": 0.0}
    R, d_in, d_out = case["rows"], case["d_in"], case["d_out"]
    x = size[case["h"]] * d_in + 4 * d_out if case["op"] == "in8" else 4 * d_in + size[case["h"]] * d_out
    return {"bytes": d_out * d_in * (1 + 1 / BLOCK) + float(R * x), "flops": 2.0 * R * d_in * d_out}


# --------------------------------------------------------------------------------------------- in 64 bits
def _exact_mass(s):
    case = s["case"]
    q, T = s["q"].double(), case["rows"]
    out = case["decay"] * s["prior"].double()
    for lib in range(case["n_lib"]):
        mine = slice(lib * T, (lib + 1) * T)
        idx, wk = s["idx"][mine].long(), s["wk"][mine].double()
        for c in range(s["page_of"].shape[1]):
            weight = (wk * (idx == c)).sum(1)
            reads = weight.nonzero().view(-1)
            if reads.numel():
                n, p = int(s["n_valid"][lib, c]), int(s["page_of"][lib, c])
                a = torch.softmax(READ_TEMP * (q[mine][reads] @ s["slots"][p, :n].double().t()), -1)
                out[p, :n] += weight[reads] @ a
    return out


def _exact_evict(s):
    case = s["case"]
    table, valid, mass = s["page_of"].tolist(), s["n_valid"].tolist(), s["mass"].double().tolist()
    P, M = len(mass), case["new_rows"]
    rows = [0] * P
    for pages, counts in zip(table, valid):
        for p, n in zip(pages, counts):
            rows[p] = max(rows[p], n)
    ranked = [sorted(range(rows[p]), key=lambda i: (-mass[p][i], i)) for p in range(P)]
    if case["per_library"]:
        stays = [set(r[:1]) for r in ranked]
        first = [set(r[:1]) for r in ranked]
        for lib, (pages, counts) in enumerate(zip(table, valid)):
            budget = int(s["keep"][lib])
            others = []
            for c, (p, n) in enumerate(zip(pages, counts)):
                budget -= sum(i < n for i in first[p])
                others += [(-mass[p][i], c, i, p) for i in ranked[p][1:M] if i < n]
            for _, _, i, p in sorted(others)[: max(0, budget)]:
                stays[p].add(i)
    else:
        most = [0] * P
        for pages, keeps in zip(table, s["keep"].tolist()):
            for p, k in zip(pages, keeps):
                most[p] = max(most[p], k)
        stays = [set(r[: min(max(1, most[p]), M)]) for p, r in enumerate(ranked)]
    left = [[sum(i < n for i in stays[p]) for p, n in zip(pages, counts)] for pages, counts in zip(table, valid)]
    kept = torch.full((P, M), -1, dtype=torch.int32)
    for p in range(P):
        kept[p, : len(stays[p])] = torch.tensor(sorted(stays[p]), dtype=torch.int32)
    kept = kept.to("cuda")
    there, src = kept >= 0, kept.clamp(min=0).long()
    new_mass = torch.where(there, torch.gather(s["mass"].double(), 1, src), 0.0)
    pools = []
    for pool in s["pools"]:
        new = torch.zeros(P, M, pool.shape[2], dtype=torch.float64, device="cuda")
        p, j = there.nonzero(as_tuple=True)
        new[p, j] = pool[p, src[p, j]].double()
        pools.append(new)
    return [torch.tensor(left, dtype=torch.int32, device="cuda"), new_mass, kept] + pools


def _rounded(x):
    """x [n, k] float64 in blocks of 128 columns as the 8-bit format holds them: three bits behind the leading one, down to
    2^-9, after a power of two that brings the largest of the block to at most 448."""
    n, k = x.shape
    x = torch.nn.functional.pad(x, (0, -k % BLOCK)).view(n, -1, BLOCK)
    top = x.abs().amax(-1, keepdim=True)
    two = torch.exp2(torch.ceil(torch.log2(top.clamp(min=1e-300) / E4M3_MAX)))
    two = torch.where(top > E4M3_MAX * two, two * 2, torch.where(top <= E4M3_MAX * two / 2, two / 2, two))
    two = torch.where(top > 0, two.clamp(2.0 ** -127, 2.0 ** 127), 1.0)
    v = x / two
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
    return (torch.round(v / step) * step * two).view(n, -1)[:, :k]


def _exact_project(s):
    case = s["case"]
    x = (s["h"] if case["op"] == "in8" else s["r"]).double()
    scale = 2.0 ** (s["w_scale"].double() - 127.0)
    w = (s["w8"].double() * scale.repeat_interleave(BLOCK, 1))[:, : case["d_in"]]
    y = torch.einsum("rk,nk->rn", _rounded(x), w)
    if case["op"] == "out8":
        return y * s["gate"].double()[:, None]
    y = y / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + EPS) + s["b"].double()
    return y / (y.norm(dim=-1, keepdim=True) + EPS)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "read_mass":
        return _exact_mass(s)
    return _exact_evict(s) if case["op"] == "pages_evict" else _exact_project(s)
