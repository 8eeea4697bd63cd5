"""The decoding operators this framework is measured on: a beam search's step, its hypotheses' pages in a cache, and attention
over the pages that a cheap score keeps.

  listed()               the named cases
  draw(rng)              one more case of the same ranges
  prepare(case, seed)    what a program holds before the call, on the GPU, from the seed alone
  run(state)             one pass: the plain form in 32 bits (64 next to a border), or (own) the framework's operators
  work(case)             the bytes and operations a pass cannot do without
  exact(case, seed)      run's outputs from the definitions in 64 bits

Beam step: a beam's candidates have total = score + logit - log sum exp logits (a finished beam: its score, for the padding
token alone) and rank = total / max(length, 1)^alpha, the length one more than the beam's (a finished one's its own). The
`keep` best of a sequence's beams, ties to the lower beam, then the larger logit, then the lower token; then the beams' states
in the chosen order.

Pages: a pool counts for each page the table entries that hold it. A fork makes row s of a table what row parents[s] was
(below 0: empty). Room for `new` more tokens gives every position behind the length a page of the row's own: where there is
none, or one that others hold, the lowest free page, in the order of rows; the rows before the length are copied, and where
all that hold a page ask for room, the first of them keeps it. A move packs the pages in use, in order, into another cache.

Bounds: the smallest and largest of each element of a page's keys, rounded outward to bfloat16, for the pages that new tokens
complete.

Sparse attention: a page's score for a token and cached head is the sum over the group's query heads and the elements of
max(q * smallest, q * largest). Of the pages that hold positions up to the token's own, the first and the last ones and the
best others are kept, `keep` in all (ties to the lower page), and the softmax runs over their keys."""

import math
import os
import sys
from types import SimpleNamespace

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PACKAGE = os.path.join(ROOT, "n-gram-hinted-lm_amd")

VOCAB = 50257
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
CODES = {"int8": torch.int8, "fp8": torch.float8_e4m3fn, "bf16": torch.bfloat16, "fp16": torch.float16}
TOP = {"int8": 127.0, "fp8": 448.0}


def listed():
    return [
        # one prompt's four hypotheses, the smallest step of a search
        {"name": "beam_4_one", "kind": "beam", "seqs": 1, "beams": 4, "keep": 4, "vocab": VOCAB, "dtype": "bf16",
         "alpha": 0.0, "ended": 0.0, "state": 4096},
        # a serving batch: 64 prompts of eight hypotheses, some of them finished, lengths normalised, recurrent states
        {"name": "beam_8_x64", "kind": "beam", "seqs": 64, "beams": 8, "keep": 8, "vocab": VOCAB, "dtype": "bf16",
         "alpha": 0.6, "ended": 0.2, "state": 65536},
        # a wide search in 32 bits over a larger vocabulary of odd size, twice as many candidates kept as there are beams
        {"name": "beam_32_wide", "kind": "beam", "seqs": 8, "beams": 32, "keep": 64, "vocab": 100003, "dtype": "fp32",
         "alpha": 1.0, "ended": 0.1, "state": 1001},
        # one prompt's hypotheses reordered, each with room for its next token
        {"name": "fork_4_one", "kind": "fork", "seqs": 1, "beams": 4, "context": 1000, "page": 16, "heads": 8, "dim": 128,
         "codes": "int8", "new": 1},
        # the serving batch's
        {"name": "fork_8_x64", "kind": "fork", "seqs": 64, "beams": 8, "context": 4096, "page": 64, "heads": 8, "dim": 128,
         "codes": "int8", "new": 1},
        # a cache in 16 bits of which a third of the pages is in use, packed into another one
        {"name": "move_bf16", "kind": "move", "pages": 8192, "rows": 64, "page": 64, "heads": 8, "dim": 128,
         "codes": "bf16"},
        # decoding: every sequence's token is the last of its page
        {"name": "bounds_x64", "kind": "bounds", "seqs": 64, "new": 1, "context": 2047, "page": 64, "heads": 8, "dim": 128,
         "codes": "int8", "ragged": False},
        # a ragged batch of prompts' chunks
        {"name": "bounds_chunks", "kind": "bounds", "seqs": 9, "new": 4001, "context": 5000, "page": 32, "heads": 8,
         "dim": 128, "codes": "fp8", "ragged": True},
        # the smallest step: one sequence, one token
        {"name": "sparse_one_5k", "kind": "sparse", "seqs": 1, "width": 1, "heads": 8, "group": 4, "dim": 128, "page": 16,
         "codes": "int8", "dtype": "bf16", "context": 5000, "keep": 32, "first": 1, "last": 2, "ragged": False,
         "lse": False},
        # a serving batch's step over ragged long contexts
        {"name": "sparse_32_x32k", "kind": "sparse", "seqs": 32, "width": 1, "heads": 8, "group": 4, "dim": 128, "page": 64,
         "codes": "int8", "dtype": "bf16", "context": 32768, "keep": 32, "first": 1, "last": 2, "ragged": True,
         "lse": False},
        # the longest contexts, four drafted tokens in a chain
        {"name": "sparse_512k", "kind": "sparse", "seqs": 2, "width": 4, "heads": 8, "group": 4, "dim": 128, "page": 64,
         "codes": "fp8", "dtype": "bf16", "context": 524288, "keep": 64, "first": 1, "last": 2, "ragged": False,
         "lse": True},
        # a prompt's next chunk, every token over pages of its own choice, a head size that is no power of two
        {"name": "sparse_chunk_1k", "kind": "sparse", "seqs": 1, "width": 1024, "heads": 5, "group": 3, "dim": 80,
         "page": 32, "codes": "fp16", "dtype": "fp16", "context": 16001, "keep": 24, "first": 1, "last": 2, "ragged": False,
         "lse": True},
    ]


def draw(rng):
    def log(lo, hi):
        return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    kind = rng.choice(("beam", "beam", "fork", "move", "bounds", "sparse", "sparse", "sparse"))
    if kind == "beam":
        beams = log(1, 32)
        return _within({"kind": kind, "seqs": log(1, 64), "beams": beams, "keep": beams * rng.choice((1, 1, 2)),
                        "vocab": log(1000, 131072), "dtype": rng.choice(("bf16", "bf16", "fp16", "fp32")),
                        "alpha": rng.choice((0.0, 0.6, 1.0)), "ended": rng.choice((0.0, 0.2)),
                        "state": log(64, 65536)}, "seqs", "state")
    cache = {"page": rng.choice((16, 32, 64, 128, 256)), "heads": rng.choice((1, 2, 3, 4, 5, 8, 8, 12, 16)),
             "dim": rng.choice((64, 64, 80, 96, 128, 128, 192, 256)), "codes": rng.choice(("int8", "fp8", "bf16", "fp16"))}
    if kind == "fork":
        return _within({"kind": kind, "seqs": log(1, 64), "beams": log(1, 16), "context": log(1, 8192), **cache,
                        "new": rng.choice((1, 1, log(2, 300)))}, "seqs", "context")
    if kind == "move":
        return _within({"kind": kind, "pages": log(16, 8192), "rows": log(1, 64), **cache}, "pages")
    if kind == "bounds":
        new, page = rng.choice((1, log(2, 4096))), cache["page"]
        ragged = new >= page and rng.random() < 0.7
        context = log(1, 8192)
        if new < page:  # every sequence's tokens end a page
            context = -(-(context + new) // page) * page - new
        return _within({"kind": kind, "seqs": log(1, 64), "new": new, "context": context, **cache, "ragged": ragged}, "seqs")
    keep = log(3, 64)
    first = rng.choice((0, 1, 1, 2)) if keep > 4 else 0
    return _within({"kind": kind, "seqs": log(1, 32), "width": rng.choice((1, 1, log(2, 512))), **cache,
                    "group": rng.choice((1, 2, 3, 4, 4, 8)),
                    "dtype": cache["codes"] if cache["codes"] in ("bf16", "fp16") else rng.choice(("bf16", "fp16")),
                    "context": log(1, 524288), "keep": keep, "first": first, "last": rng.choice((1, 2)),
                    "ragged": rng.random() < 0.6, "lse": rng.random() < 0.5}, "seqs", "width", "context")


def _within(case, *sizes):
    """The case with its sizes halved in turn until it costs no more than the largest listed one of its kind."""
    top = [work(c) for c in listed() if c["kind"] == case["kind"]]
    limit = {k: max(w[k] for w in top) for k in ("bytes", "flops")}
    limit["held"] = max(_held(c) for c in listed() if c["kind"] == case["kind"])
    limit["rows"] = max(_rows(c) for c in listed() if c["kind"] == case["kind"])
    i = 0
    while any(v > limit[k] for k, v in (*work(case).items(), ("held", _held(case)), ("rows", _rows(case)))):
        size = sizes[i % len(sizes)]
        case[size] = max(1, case[size] // 2)
        i += 1
    return case


def _rows(case):
    """The choices of pages that a case makes."""
    return case["seqs"] * case["width"] * case["heads"] if case["kind"] == "sparse" else 0


def _held(case):
    """Bytes of the cache that a case holds."""
    if case["kind"] == "beam":
        return 0
    token = case["heads"] * _padded(case["dim"]) * (2 if case["codes"] in ("bf16", "fp16") else 1)
    if case["kind"] == "move":
        return case["pages"] * case["page"] * token
    tokens = case["context"] + case.get("new", case.get("width", 0)) + case["page"] * case.get("beams", 1)
    return case["seqs"] * tokens * token


# ---------------------------------------------------------------------------------------------------------- inputs


def _lengths(case):
    """The sequences' cached lengths: from the case alone. Ragged: down to a quarter of the context; where there are three
    sequences or more, the first has no context."""
    B, C = case["seqs"], case["context"]
    if not case["ragged"]:
        return [C] * B
    lengths = [C - (b * 7919) % (3 * C // 4 + 1) for b in range(B)]
    if B >= 3:
        lengths[0] = 0
    return lengths


def _widths(case):
    B, T = case["seqs"], case["width"]
    return [T - (b * 5) % (T // 2 + 1) for b in range(B)] if case["ragged"] else [T] * B


def _padded(dim):
    return (dim + 63) // 64 * 64


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _bits(t):
    """The codes as integers of their size: elementary indexing has no 8-bit floats."""
    return t.view({1: torch.uint8, 2: torch.int16}[t.element_size()])


def _stored(heads, pages, page, dim, codes, g, apart=0.0):
    """A filled cache: codes and scales of random rows, the rows of a page around a middle of their own."""
    held = torch.zeros((pages, heads, page, _padded(dim)), dtype=torch.uint8 if codes in TOP else CODES[codes], device="cuda")
    held = held.view(CODES[codes])
    scales = torch.zeros((pages, heads, page), device="cuda") if codes in TOP else None
    step = max(1, (1 << 28) // (heads * page * dim))
    for p in range(0, pages, step):  # some pages at a time: the rows in 32 bits are up to four times the cache
        n = min(step, pages - p)
        x = torch.randn((n, heads, page, dim), generator=g, device="cuda")
        x += apart * torch.randn((n, heads, 1, dim), generator=g, device="cuda")
        if scales is None:
            held[p:p + n, ..., :dim] = x.to(held.dtype)
            continue
        a = x.abs().amax(-1)
        x *= (TOP[codes] / a)[..., None]
        _bits(held)[p:p + n, ..., :dim] = _bits((x.round_() if codes == "int8" else x).to(held.dtype))
        scales[p:p + n] = a / TOP[codes]
    return held, scales


def _framework(module):
    if PACKAGE not in sys.path:
        sys.path.insert(0, PACKAGE)
    import importlib

    return importlib.import_module("ngram_amd." + module)


def prepare(case, seed):
    return {"beam": _prepare_beam, "fork": _prepare_fork, "move": _prepare_move, "bounds": _prepare_bounds,
            "sparse": _prepare_sparse}[case["kind"]](case, seed)


def _prepare_beam(case, seed):
    """Logits of a spread at which a few tokens take most of the weight, beams' scores of some tokens' sums, in order."""
    g = _generator(seed)
    B, W, V = case["seqs"], case["beams"], case["vocab"]
    s = SimpleNamespace(kind="beam", keep=case["keep"], alpha=case["alpha"], end=V - 1)
    s.logits = (torch.randn((B, W, V), generator=g, device="cuda") * 3).to(DTYPES[case["dtype"]])
    s.scores = -(torch.rand((B, W), generator=g, device="cuda") * 4).cumsum(1) - 10
    s.lengths = torch.randint(1, 40, (B, W), generator=g, device="cuda").int()
    s.finished = torch.rand((B, W), generator=g, device="cuda") < case["ended"]
    s.state = torch.randn((B * W, case["state"]), generator=g, device="cuda")
    if own:
        beam = _framework("beam")
        s.step, s.reorder = beam.beam_step, beam.reorder
    return s


def _prepare_fork(case, seed):
    """Each sequence's beams hold its prompt's pages in common and one to three of their own, lengths are those of the beams'
    common step; a parent has more children the lower its beam; every sixteenth sequence has ended and leaves."""
    g = _generator(seed)
    B, W, P, C, new = case["seqs"], case["beams"], case["page"], case["context"], case["new"]
    s = SimpleNamespace(kind="fork", dim=case["dim"], page=P, new=new)
    lengths = [max(1, C - (b * 7919) % (C // 2 + 1)) for b in range(B)]
    width = -(-(max(lengths) + new) // P) + 1
    own_pages = (torch.rand((B, W), generator=g, device="cuda") * 3).long().cpu().numpy()
    table = torch.full((B * W, width), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(lengths):
        used = -(-n // P)
        for w in range(W):
            common = max(0, used - 1 - int(own_pages[b, w])) if w else 0
            table[b * W + w, :common] = table[b * W, :common]
            table[b * W + w, common:used] = torch.arange(at, at + used - common, dtype=torch.int32)
            at += used - common
    pages = sum(-(-n // P) + 3 * (W - 1) for n in lengths) + B * W * (-(-new // P) + 2)  # (the inputs' seed aside)
    order = torch.randperm(pages, generator=g, device="cuda").int()
    table = table.cuda()
    s.table = torch.where(table >= 0, order[table.clamp(min=0)], table)
    s.lengths = torch.tensor(lengths, dtype=torch.int32).repeat_interleave(W).cuda()
    child = (torch.rand((B, W), generator=g, device="cuda") ** 2 * W).long() + torch.arange(B, device="cuda")[:, None] * W
    child[15::16] = -1
    s.parents = child.reshape(-1)
    s.k, s.k_scale = _stored(case["heads"], pages, P, s.dim, case["codes"], g)
    s.v, s.v_scale = _stored(case["heads"], pages, P, s.dim, case["codes"], g)
    if own:
        s.cache = _framework("kvcache").KVCache(s.k, s.v, s.k_scale, s.v_scale, dim=s.dim)
        s.pool = _framework("pages").PagePool(s.cache)
        s.pool.hold(s.table)
    else:
        s.refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
        held = s.table[s.table >= 0].long()
        s.refs.index_add_(0, held, torch.ones_like(held, dtype=torch.int32))
    return s


def _prepare_move(case, seed):
    """A third of the pages in use, by rows of even shares of them in a random order; the cache moved to has just room."""
    g = _generator(seed)
    N, S, P, H = case["pages"], case["rows"], case["page"], case["heads"]
    s = SimpleNamespace(kind="move", dim=case["dim"])
    live = max(1, N // 3)
    width = -(-live // S)
    table = torch.full((S * width,), -1, dtype=torch.int32, device="cuda")
    table[:live] = torch.randperm(N, generator=g, device="cuda")[:live].int()
    s.table = table.view(width, S).t().contiguous()
    s.k, s.k_scale = _stored(H, N, P, s.dim, case["codes"], g)
    s.v, s.v_scale = _stored(H, N, P, s.dim, case["codes"], g)
    room = live + 2
    s.to = [None if t is None else _zeros_like(t, room) for t in (s.k, s.v, s.k_scale, s.v_scale)]
    if own:
        KVCache, PagePool = _framework("kvcache").KVCache, _framework("pages").PagePool
        s.cache = KVCache(s.k, s.v, s.k_scale, s.v_scale, dim=s.dim)
        s.into = PagePool(KVCache(*s.to, dim=s.dim))
        s.pool = PagePool(s.cache)
        s.pool.hold(s.table)
    else:
        s.refs = torch.zeros(N, dtype=torch.int32, device="cuda")
        held = s.table[s.table >= 0].long()
        s.refs.index_add_(0, held, torch.ones_like(held, dtype=torch.int32))
    return s


def _zeros_like(t, pages):
    shape = (pages, *t.shape[1:])
    if t.element_size() == 1:
        return torch.zeros(shape, dtype=torch.uint8, device="cuda").view(t.dtype)
    return torch.zeros(shape, dtype=t.dtype, device="cuda")


def _tables(lengths, widths, page, g):
    """Page tables over pages in a random order, unused entries -1; the cache's pages."""
    used = [-(-(n + t) // page) for n, t in zip(lengths, widths)]
    pages = sum(used) + 2
    order = torch.randperm(pages, generator=g, device="cuda").int()
    table = torch.full((len(used), max(used)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, m in enumerate(used):
        table[b, :m] = order[at:at + m]
        at += m
    return table, pages


def _prepare_bounds(case, seed):
    g = _generator(seed)
    B, new, P, H = case["seqs"], case["new"], case["page"], case["heads"]
    s = SimpleNamespace(kind="bounds", dim=case["dim"], new=new, page=P)
    lengths = _lengths(case)
    s.table, pages = _tables(lengths, [new] * B, P, g)
    s.start = torch.tensor(lengths, dtype=torch.int32).cuda()
    s.k, s.k_scale = _stored(H, pages, P, s.dim, case["codes"], g)
    s.bounds = torch.randn((pages, H, 2, _padded(s.dim)), generator=g, device="cuda").bfloat16()
    if own:
        s.cache = _framework("kvcache").KVCache(s.k, s.k, s.k_scale, s.k_scale, dim=s.dim)
        s.index = _framework("sparse").PageBounds(s.cache, s.bounds)
    return s


def _prepare_sparse(case, seed):
    """Keys of a page lie around a middle of their own, queries are of twice the keys' size (so that the softmax is not flat)."""
    g = _generator(seed)
    B, T, H, G, D, P = (case[k] for k in ("seqs", "width", "heads", "group", "dim", "page"))
    lengths, widths = _lengths(case), _widths(case)
    s = SimpleNamespace(kind="sparse", dim=D, heads=H, page=P, keep=case["keep"], first=case["first"], last=case["last"],
                        lse=case["lse"], scale=1 / math.sqrt(D), dtype=DTYPES[case["dtype"]])
    s.table, pages = _tables(lengths, [T] * B, P, g)
    s.lengths = torch.tensor(lengths, dtype=torch.int32).cuda()
    s.widths = torch.tensor(widths, dtype=torch.int32).cuda() if case["ragged"] else None
    s.k, s.k_scale = _stored(H, pages, P, D, case["codes"], g, 0.7)
    s.v, s.v_scale = _stored(H, pages, P, D, case["codes"], g)
    s.bounds = torch.zeros((pages, H, 2, _padded(D)), dtype=torch.bfloat16, device="cuda")
    step = max(1, (1 << 28) // (H * P * D))
    for p in range(0, pages, step):
        s.bounds[p:p + step, ..., :D] = _plain_bounds(_plain_values(s.k[p:p + step], None if s.k_scale is None else
                                                                    s.k_scale[p:p + step], D))
    s.q = (torch.randn((B, T, H * G, D), generator=g, device="cuda") * 2).to(s.dtype)
    if own:
        s.cache = _framework("kvcache").KVCache(s.k, s.v, s.k_scale, s.v_scale, dim=D)
        sparse = _framework("sparse")
        s.index, s.attend = sparse.PageBounds(s.cache, s.bounds), sparse.sparse_attention
    return s


# ------------------------------------------------------------------------------------------------------------- run


def run(state):
    return {"beam": _run_beam, "fork": _run_fork, "move": _run_move, "bounds": _run_bounds,
            "sparse": _run_sparse}[state.kind](state)


def _run_beam(s):
    if own:
        step = s.step(s.logits, s.scores, s.lengths, s.finished, keep=s.keep, end=s.end, alpha=s.alpha)
        return [*step, s.reorder(s.state, step.parents)]
    B, W, V = s.logits.shape
    x = s.logits.double()  # totals of different beams lie next to each other
    top = x.amax(-1, keepdim=True)
    total = s.scores.double()[..., None] + (x - ((x - top).exp().sum(-1, keepdim=True).log() + top))
    del x, top
    total.masked_fill_(s.finished[..., None], -math.inf)
    total[..., s.end] = torch.where(s.finished, s.scores.double(), total[..., s.end])
    length = s.lengths + torch.where(s.finished, 0, 1)
    rank = (total / length.double().clamp(min=1)[..., None] ** s.alpha).reshape(B, -1)
    rank = torch.where(rank == rank, rank, -math.inf)
    at = rank.sort(dim=-1, descending=True, stable=True).indices[:, :s.keep]
    scores = torch.where(rank == -math.inf, -math.inf, total.reshape(B, -1)).gather(1, at).float()
    beam, token = at // V, at % V
    finished = s.finished.gather(1, beam) | (token == s.end)
    parents = beam + torch.arange(B, device=at.device)[:, None] * W
    return [scores, parents, token, finished, length.gather(1, beam), s.state[parents.reshape(-1)]]


def _run_fork(s):
    if own:
        s.pool.fork(s.table, s.lengths, s.parents)
        slots = s.pool.reserve(s.table, s.lengths, s.new)
        return [slots, s.table, s.lengths, s.pool.refs, *(t for t in (s.k, s.v, s.k_scale, s.v_scale) if t is not None)]
    P, (S, width) = s.page, s.table.shape
    # the fork
    stays = s.parents >= 0
    children = torch.zeros(S, dtype=torch.int32, device=s.table.device)
    children.index_add_(0, s.parents.clamp(min=0), stays.int())
    held = s.table >= 0
    s.refs.index_add_(0, s.table.clamp(min=0).reshape(-1).long(), torch.where(held, children[:, None] - 1, 0).int().reshape(-1))
    s.table.copy_(torch.where(stays[:, None], s.table[s.parents.clamp(min=0)], -1))
    s.lengths.copy_(torch.where(stays, s.lengths[s.parents.clamp(min=0)], 0))
    # the pages that hold the next positions
    m = (s.new - 1) // P + 2
    column = (s.lengths // P)[:, None] + torch.arange(m, device=s.table.device)
    asked = (column * P < s.lengths[:, None] + s.new) & (column < width)
    at = column.clamp(max=width - 1).long()
    page = s.table.gather(1, at)
    held = asked & (page >= 0)
    flat, place = page.clamp(min=0).reshape(-1).long(), torch.arange(S * m, device=s.table.device)
    askers = torch.zeros_like(s.refs).index_add_(0, flat, held.reshape(-1).int())
    order = torch.where(held.reshape(-1), place, S * m)
    first = torch.full(s.refs.shape, S * m, device=s.table.device).scatter_reduce_(0, flat, order, "amin")
    alone = (s.refs[flat] == askers[flat]) & (first[flat] == place)
    wanted = asked.reshape(-1) & ~(held.reshape(-1) & alone)
    # the lowest free ones in order, the rows before the length copied
    free = s.refs == 0
    lowest = free.logical_not().int().sort(stable=True).indices
    rank = wanted.cumsum(0) - 1
    got = wanted & (rank < free.sum())
    new = lowest[rank.clamp(0, s.refs.shape[0] - 1)]
    left = got & held.reshape(-1)
    s.refs.index_add_(0, flat, -left.int())
    s.refs[new[got]] = 1
    behind = (s.lengths[:, None] - column * P).reshape(-1)
    copied = left & (behind > 0)
    a, b, n = flat[copied], new[copied], behind[copied]
    rows = torch.arange(P, device=s.table.device) < n[:, None, None]
    for t in (s.k, s.v):
        _bits(t)[b] = torch.where(rows[..., None], _bits(t)[a], _bits(t)[b])
    for t in (s.k_scale, s.v_scale):
        if t is not None:
            t[b] = torch.where(rows, t[a], t[b])
    page = torch.where(got, new, page.reshape(-1)).int()
    row = torch.arange(S, device=s.table.device)[:, None].expand(S, m).reshape(-1)
    s.table[row[got], at.reshape(-1)[got]] = page[got]
    fine = (asked.reshape(-1) & (got | ~wanted)).reshape(S, m)
    where = s.lengths[:, None].long() + torch.arange(s.new, device=s.table.device)
    j = where // P - (s.lengths // P)[:, None]
    slots = torch.where(fine.gather(1, j), page.reshape(S, m).gather(1, j).long() * P + where % P, -1)
    return [slots, s.table, s.lengths, s.refs, *(t for t in (s.k, s.v, s.k_scale, s.v_scale) if t is not None)]


def _run_move(s):
    if own:
        table = s.pool.move(s.table, s.into)
        return [table, s.into.refs, *(t for t in s.to if t is not None)]
    live = s.refs > 0
    to = torch.where(live, live.cumsum(0) - 1, -1)
    pages = live.nonzero()[:, 0]
    refs = torch.zeros(s.to[0].shape[0], dtype=torch.int32, device=s.refs.device)
    refs[:pages.shape[0]] = s.refs[pages]
    for a, b in zip((s.k, s.v, s.k_scale, s.v_scale), s.to):
        if a is not None and a.element_size() < 4:
            _bits(b)[:pages.shape[0]] = _bits(a)[pages]
        elif a is not None:
            b[:pages.shape[0]] = a[pages]
    table = torch.where(s.table >= 0, to[s.table.clamp(min=0).long()], -1).int()
    return [table, refs, *(t for t in s.to if t is not None)]


def _plain_values(codes, scales, dim):
    x = codes[..., :dim].float()
    return x if scales is None else x * scales[..., None]


def _plain_bounds(x):
    """x [..., page, dim]: its smallest and largest rows [..., 2, dim], in bfloat16 away from each other."""
    lo, hi = x.amin(-2), x.amax(-2)

    def cut(v, away):  # towards zero, one step further where that is not the way and something was cut
        bits = v.view(torch.int32)
        near = bits & -65536
        far = torch.where(away & (bits != near), near + 65536, near)
        return torch.where(v == v, far.view(torch.float32), v)

    return torch.stack([cut(lo, lo < 0), cut(hi, hi > 0)], -2).bfloat16()


def _run_bounds(s):
    if own:
        s.index.update(s.table, s.start, s.new)
        return s.bounds
    P, width = s.page, s.table.shape[1]
    m = (s.new - 1) // P + 2
    column = (s.start // P)[:, None] + torch.arange(m, device=s.table.device)
    whole = ((column + 1) * P <= s.start[:, None] + s.new) & (column < width)
    page = s.table.gather(1, column.clamp(max=width - 1).long())[whole].long()
    codes = _bits(s.k)[page].view(s.k.dtype)
    s.bounds[page, ..., :s.dim] = _plain_bounds(_plain_values(codes, None if s.k_scale is None else s.k_scale[page], s.dim))
    s.bounds[page, ..., s.dim:] = 0
    return s.bounds


def _run_sparse(s):
    if own:
        return s.attend(s.q, s.cache, s.index, s.table, s.lengths, s.keep, s.widths, first=s.first, last=s.last,
                        scale=s.scale, return_lse=s.lse, return_pages=True)
    B, T, Hq, D = s.q.shape
    H, P, width = s.heads, s.page, s.table.shape[1]
    dev = s.q.device
    q = s.q.view(B, T, H, Hq // H, D)
    used = torch.arange(T, device=dev) < (torch.full_like(s.lengths, T) if s.widths is None else s.widths)[:, None]  # [B, T]
    place = s.lengths[:, None] + torch.arange(T, device=dev)
    seen = place // P + 1  # pages a token sees
    # the scores, in 64 bits: they lie next to each other where the last page kept is chosen
    up = q.double().clamp(min=0).sum(3).transpose(1, 2).contiguous()  # [B, H, T, D]
    down = q.double().clamp(max=0).sum(3).transpose(1, 2).contiguous()
    bounds = s.bounds[s.table.clamp(min=0).long()][..., :D].permute(0, 2, 3, 4, 1)  # [B, H, 2, D, width]
    score = torch.matmul(down, bounds[:, :, 0].double().contiguous())
    score += torch.matmul(up, bounds[:, :, 1].double().contiguous())  # [B, H, T, width]
    del bounds
    page, n = torch.arange(width, device=dev), seen[:, None, :, None]
    score.masked_fill_((page < s.first) | (page >= n - s.last), math.inf)
    score.masked_fill_(page >= n, -math.inf)
    keep = min(s.keep, width)
    at = score.sort(dim=-1, descending=True, stable=True).indices[..., :keep]
    at = torch.where(at < n, at, width).sort(dim=-1).values  # ascending, what there is not at the end
    kept = at < n
    del score
    pages = s.table[:, None, None].expand(B, H, T, width).gather(-1, at.clamp(max=width - 1)).long()
    h = torch.arange(H, device=dev)[None, :, None, None]
    where = (at[..., None] * P + torch.arange(P, device=dev)).reshape(B, H, T, -1)
    sees = (where <= place[:, None, :, None]) & used[:, None, :, None]
    k = _plain_rows(s.k, s.k_scale, pages, h, D)  # [B, H, T, keep * P, D]
    a = (torch.matmul(q.transpose(1, 2).float().contiguous(), k.transpose(3, 4).contiguous()) * s.scale)
    del k
    a.masked_fill_(~(sees & kept.repeat_interleave(P, -1))[:, :, :, None], -math.inf)  # [B, H, T, G, keep * P]
    top = a.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    p = a.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, _plain_rows(s.v, s.v_scale, pages, h, D))
    out = torch.where(total > 0, out / total, 0.0).transpose(1, 2).reshape(B, T, Hq, D).to(s.dtype)
    lse = (total.log() + top)[..., 0].transpose(1, 2).reshape(B, T, Hq)
    chosen = torch.where(kept & used[:, None, :, None], at, -1).transpose(1, 2).int()  # [B, T, H, keep]
    if keep < s.keep:
        chosen = torch.cat([chosen, torch.full((B, T, H, s.keep - keep), -1, dtype=torch.int32, device=dev)], -1)
    return [out, lse, chosen] if s.lse else [out, chosen]


def _plain_rows(held, scales, pages, h, dim):
    x = _bits(held)[pages, h].view(held.dtype)[..., :dim].float()  # [B, H, T, keep, P, D]
    if scales is not None:
        x *= scales[pages, h][..., None]
    return x.reshape(*x.shape[:3], -1, dim)


# ------------------------------------------------------------------------------------------------------------ work


def work(case):
    if case["kind"] == "beam":
        B, W, V, K = case["seqs"], case["beams"], case["vocab"], case["keep"]
        size = 4 if case["dtype"] == "fp32" else 2
        alive = B * W * (1 - case["ended"])
        return {"bytes": alive * V * size + 2 * B * K * case["state"] * 4 + B * (9 * W + 25 * K), "flops": 4.0 * alive * V}
    H, D, P = case["heads"], case["dim"], case["page"]
    code = 2 if case["codes"] in ("bf16", "fp16") else 1
    key = H * (D * code + (4 if code == 1 else 0))  # a token's keys
    if case["kind"] == "fork":
        S, C = case["seqs"] * case["beams"], case["context"]
        entries = S * (C // P + 1)
        copied = S * (1 - 1 / case["beams"]) * 0.4 * min(C, P // 2)  # the second and later children's pages, half full
        return {"bytes": 8 * entries + 8 * S * (2 + case["new"]) + 4 * copied * key, "flops": 1.0 * entries}
    if case["kind"] == "move":
        live = max(1, case["pages"] // 3)
        return {"bytes": 4 * live * P * key + 8 * case["pages"], "flops": 1.0 * case["pages"]}
    if case["kind"] == "bounds":
        whole = sum((n + case["new"]) // P - n // P for n in _lengths(case))
        return {"bytes": whole * (P * key + 4 * H * D) + 4 * whole + 1, "flops": 3.0 * whole * P * H * D + 1}
    G, K = case["group"], case["keep"]
    bytes_ = flops = 1.0
    for n, w in zip(_lengths(case), _widths(case)):
        pages = -(-(n + w) // P)
        kept = min(K, pages)
        read = pages if w == 0 else pages * (1 - (1 - kept / pages) ** w)  # what w tokens keep that choose apart
        scored = pages if pages > K else 0
        bytes_ += H * 4 * D * scored + 2 * read * P * key + 4 * case["width"] * H * G * D + 4 * case["width"] * H * K
        flops += w * H * (4.0 * D * scored + 4.0 * G * D * min(kept * P, n + w))
    return {"bytes": bytes_, "flops": flops}


# ----------------------------------------------------------------------------------------------------------- exact


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    return {"beam": _exact_beam, "fork": _exact_fork, "move": _exact_move, "bounds": _exact_bounds,
            "sparse": _exact_sparse}[case["kind"]](s)


def _exact_beam(s):
    B, W, V = s.logits.shape
    out = [[] for _ in range(5)]
    for b in range(B):
        ended, length = s.finished[b].tolist(), s.lengths[b].tolist()
        best = []  # (-rank, beam, place in the beam's order, total, token)
        for w in range(W):
            if ended[w]:
                total = float(s.scores[b, w])
                best.append((-total / max(length[w], 1) ** s.alpha, w, 0, total, s.end))
                continue
            p = torch.log_softmax(s.logits[b, w].double(), 0)
            order = torch.argsort(s.logits[b, w].float(), descending=True, stable=True)[:s.keep]
            for i, (t, lp) in enumerate(zip(order.tolist(), p[order].tolist())):
                total = float(s.scores[b, w]) + lp
                best.append((-total / (length[w] + 1) ** s.alpha, w, i, total, t))
        best.sort()
        best = best[:s.keep]
        taken = {x[1] * V + x[4] for x in best}
        spare = [i for i in range(2 * s.keep) if i not in taken]  # too few candidates: the lowest of what has no chance
        best += [(math.inf, i // V, 0, -math.inf, i % V) for i in spare[:s.keep - len(best)]]
        out[0].append([x[3] for x in best])
        out[1].append([b * W + x[1] for x in best])
        out[2].append([x[4] for x in best])
        out[3].append([x[4] == s.end or ended[x[1]] for x in best])
        out[4].append([length[x[1]] + (not ended[x[1]]) for x in best])
    scores = torch.tensor(out[0], dtype=torch.float64, device="cuda")
    parents, tokens = (torch.tensor(x, dtype=torch.int64, device="cuda") for x in out[1:3])
    finished = torch.tensor(out[3], dtype=torch.bool, device="cuda")
    lengths = torch.tensor(out[4], dtype=torch.int32, device="cuda")
    return [scores, parents, tokens, finished, lengths, s.state.index_select(0, parents.reshape(-1)).double()]


def _exact_fork(s):
    P, (S, width) = s.page, s.table.shape
    before, length, parents = s.table.tolist(), s.lengths.tolist(), s.parents.tolist()
    table = [list(before[p]) if p >= 0 else [-1] * width for p in parents]
    length = [length[p] if p >= 0 else 0 for p in parents]
    holders = {}
    for r in table:
        for g in r:
            if g >= 0:
                holders[g] = holders.get(g, 0) + 1
    free = [g for g in range(s.refs.shape[0]) if g not in holders]
    spans = [range(n // P, min(width, (n + s.new - 1) // P + 1)) for n in length]
    asking = {}
    for r, span in enumerate(spans):
        for c in span:
            if table[r][c] >= 0:
                asking.setdefault(table[r][c], []).append((r, c))
    keeps = {x[0] for g, x in asking.items() if len(x) == holders[g]}
    copies, refused, at = [], set(), 0
    for r, span in enumerate(spans):
        for c in span:
            g = table[r][c]
            if (r, c) in keeps:
                continue
            if at == len(free):
                refused.add((r, c))
                continue
            table[r][c] = free[at]
            at += 1
            holders[table[r][c]] = 1
            if g >= 0:
                holders[g] -= 1
                if length[r] > c * P:
                    copies.append((g, table[r][c], length[r] - c * P))
    slots = [[-1 if x // P >= width or (r, x // P) in refused else table[r][x // P] * P + x % P
              for x in range(length[r], length[r] + s.new)] for r in range(S)]
    held = [t for t in (s.k, s.v, s.k_scale, s.v_scale) if t is not None]
    for a, b, n in copies:
        for t in held:
            x = _bits(t) if t.element_size() < 4 else t
            x[b, :, :n] = x[a, :, :n]
    refs = [holders.get(g, 0) for g in range(s.refs.shape[0])]
    return [torch.tensor(slots, device="cuda"), torch.tensor(table, dtype=torch.int32, device="cuda"),
            torch.tensor(length, dtype=torch.int32, device="cuda"), torch.tensor(refs, dtype=torch.int32, device="cuda"), *held]


def _exact_move(s):
    refs = s.refs.tolist()
    used = [g for g, n in enumerate(refs) if n]
    to = {g: i for i, g in enumerate(used)}
    table = [[to.get(g, -1) for g in r] for r in s.table.tolist()]
    room = s.to[0].shape[0]
    for a, b in zip((s.k, s.v, s.k_scale, s.v_scale), s.to):
        if a is not None:
            x, y = (_bits(t) if t.element_size() < 4 else t for t in (a, b))
            y[:len(used)] = x.index_select(0, torch.tensor(used, device="cuda"))
    counts = [refs[g] for g in used] + [0] * (room - len(used))
    return [torch.tensor(table, dtype=torch.int32, device="cuda"), torch.tensor(counts, dtype=torch.int32, device="cuda"),
            *(t for t in s.to if t is not None)]


def _exact_rows(held, scales, page, h, dim):
    """The values of some pages of one head in 64 bits (their definition rounds code * scale to 32): [rows, dim]."""
    x = held[page, h].float().double()[..., :dim]
    if scales is not None:
        x = (x * scales[page, h].double()[..., None]).float().double()
    return x.reshape(-1, dim)


def _exact_bounds(s):
    P, out = s.page, s.bounds.double()
    table = s.table.tolist()
    for b, n in enumerate(s.start.tolist()):
        done = torch.tensor(table[b][n // P:min((n + s.new) // P, len(table[b]))], dtype=torch.int64, device="cuda")
        for h in range(s.k.shape[1]):
            x = _exact_rows(s.k, s.k_scale, done, h, s.dim).reshape(done.shape[0], P, s.dim)
            if not done.shape[0]:
                continue
            for i, v in enumerate((x.min(1).values, x.max(1).values)):
                step = torch.exp2(torch.frexp(v).exponent.double() - 8)  # bfloat16's at v
                out[done, h, i, :s.dim] = (torch.floor(v / step) if i == 0 else torch.ceil(v / step)) * step
                out[done, h, i, s.dim:] = 0
    return out


def _exact_sparse(s):
    import numpy

    B, T, Hq, D = s.q.shape
    G, P, K = Hq // s.heads, s.page, s.keep
    out = torch.zeros((B, T, Hq, D), device="cuda", dtype=torch.float64)
    lse = torch.full((B, T, Hq), -math.inf, device="cuda", dtype=torch.float64)
    chosen = torch.full((B, T, s.heads, K), -1, dtype=torch.int32)
    lengths = s.lengths.tolist()
    widths = [T] * B if s.widths is None else s.widths.tolist()
    for b in range(B):
        n, w = lengths[b], widths[b]
        pages = s.table[b, :-(-(n + w) // P)].long()
        for h in range(s.heads):
            q = s.q[b, :w, h * G:(h + 1) * G].double()
            lo, hi = (s.bounds[pages, h, i, :D].double() for i in (0, 1))
            score = sum(torch.where(q[:, g] > 0, q[:, g], 0.0) @ hi.T + torch.where(q[:, g] < 0, q[:, g], 0.0) @ lo.T
                        for g in range(G)).cpu().numpy()
            k, v = (_exact_rows(x, y, pages, h, D) for x, y in ((s.k, s.k_scale), (s.v, s.v_scale)))
            for t in range(w):
                m = (n + t) // P + 1
                must = {j for j in range(m) if j < s.first or j >= m - s.last}
                rest = [j for j in numpy.argsort(-score[t, :m], kind="stable")[:K + len(must)].tolist() if j not in must]
                mine = sorted(must | set(rest[:max(0, K - len(must))]))
                chosen[b, t, h, :len(mine)] = torch.tensor(mine, dtype=torch.int32)
                at = (torch.tensor(mine)[:, None] * P + torch.arange(P)).reshape(-1)
                at = at[at <= n + t].cuda()
                a = (q[t] @ k[at].T) * s.scale
                z = torch.logsumexp(a, 1)
                lse[b, t, h * G:(h + 1) * G] = z
                out[b, t, h * G:(h + 1) * G] = torch.exp(a - z[:, None]) @ v[at]
    return [out, lse, chosen.cuda()] if s.lse else [out, chosen.cuda()]
