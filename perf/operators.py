"""The model-side operators this framework is measured on: hint rows embedded and their table's gradient, a key/value
cache held in 8 bits, and attention for a tree of drafted tokens over that cache.

  listed()               the named cases
  draw(rng)              one more case of the same ranges
  prepare(case, seed)    what a program holds before the call, on the GPU, from the seed alone
  run(state)             one pass: the plain form in 32 bits, or (own) the framework's operators
  work(case)             the bytes and operations a pass cannot do without
  exact(case, seed)      run's outputs from the definitions in 64 bits

Embedding: out[n] = scale * sum over slots s with cell[n, s] > 0 and entries e with w[n, s, e] != 0 of
w[n, s, e] * table[tok[n, s, e]]; without weights a plain lookup, scale * table[tok[n]].

Cache: a token's row x of one head is held as codes and a float32 scale. With a = max |x| and M = 127 (int8) or 448 (fp8,
e4m3fn): code = x * (M / a) rounded half to even in that type, scale = a / M; in 16 bits the codes are x itself. Codes
lie in [pages, heads, page size, dim padded with zeros to a multiple of 64], scales in [pages, heads, page size]; slot p of
a token is its page * page size + its row there, and -1 is no slot (not written; read as zeros).

Tree attention: sequence b has lengths[b] cached tokens and widths[b] tree tokens at the positions behind them; tree token
i sees every cached token and tree token j where bit j of mask[b, i] is set. Rows at or past widths[b], and rows that see
nothing, are zeros (their log-sum-exp -inf)."""

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
        # one decoding step's drafted tokens: the hint rows of 16 positions
        {"name": "embed_step_16", "kind": "embed", "n": 16, "slots": 1, "entries": 8, "dim": 768, "dtype": "bf16",
         "train": False, "learned": False},
        # a training micro-batch of 64 x 1024 positions, one slot of 8 candidates, and the table's gradient
        {"name": "embed_rows_64k", "kind": "embed", "n": 65536, "slots": 1, "entries": 8, "dim": 768, "dtype": "bf16",
         "train": True, "learned": False},
        # a ragged batch, two slots, rows of odd length in 32 bits, the weights learned as well
        {"name": "embed_learned_20011", "kind": "embed", "n": 20011, "slots": 2, "entries": 8, "dim": 333,
         "dtype": "fp32", "train": True, "learned": True},
        # a training micro-batch's own tokens: a plain scaled lookup, frequent tokens' gradients summed over many rows
        {"name": "embed_tokens_128k", "kind": "embed", "n": 131072, "slots": 1, "entries": 0, "dim": 1024,
         "dtype": "bf16", "train": True, "learned": False},
        # eight sequences append one decoded token each
        {"name": "cache_append_8", "kind": "cache", "write": 8, "read": 0, "heads": 8, "dim": 128, "page": 16,
         "codes": "fp8", "dtype": "bf16", "skip": False},
        # a prompt's next chunk written, the sequence so far read back for an attention over dense keys and values
        {"name": "cache_chunk_4k", "kind": "cache", "write": 4096, "read": 32768, "heads": 8, "dim": 128, "page": 64,
         "codes": "int8", "dtype": "bf16", "skip": False},
        # packed prompts of odd sizes, some tokens without a slot, a head size that is no power of two
        {"name": "cache_ragged_fp16", "kind": "cache", "write": 5003, "read": 5003, "heads": 5, "dim": 80, "page": 16,
         "codes": "fp8", "dtype": "fp16", "skip": True},
        # the smallest step: one sequence, one token, a short context
        {"name": "tree_one_300", "kind": "tree", "seqs": 1, "width": 1, "heads": 8, "group": 4, "dim": 128, "page": 16,
         "codes": "int8", "dtype": "bf16", "context": 300, "ragged": False, "lse": False},
        # an ordinary step: eight sequences of different lengths, trees of 16 drafted tokens
        {"name": "tree_16_x8", "kind": "tree", "seqs": 8, "width": 16, "heads": 8, "group": 4, "dim": 128, "page": 64,
         "codes": "int8", "dtype": "bf16", "context": 4096, "ragged": True, "lse": False},
        # no grouping, a 16-bit cache, odd sizes, an empty context and unused tree rows
        {"name": "tree_33_mha_fp16", "kind": "tree", "seqs": 5, "width": 33, "heads": 12, "group": 1, "dim": 64,
         "page": 16, "codes": "fp16", "dtype": "fp16", "context": 1021, "ragged": True, "lse": True},
        # a serving batch: 64 sequences, small trees, long contexts
        {"name": "tree_8_x64", "kind": "tree", "seqs": 64, "width": 8, "heads": 8, "group": 4, "dim": 128, "page": 64,
         "codes": "int8", "dtype": "bf16", "context": 8192, "ragged": True, "lse": False},
        # the longest contexts under the widest tree
        {"name": "tree_64_long", "kind": "tree", "seqs": 2, "width": 64, "heads": 8, "group": 4, "dim": 128, "page": 64,
         "codes": "fp8", "dtype": "bf16", "context": 131072, "ragged": False, "lse": True},
    ]


def draw(rng):
    def log(lo, hi):
        return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    kind = rng.choice(("embed", "cache", "tree", "tree"))
    if kind == "embed":
        slots, entries = rng.choice((1, 1, 2)), rng.choice((8, 8, 4, 1, 0))
        if entries == 0:
            slots = 1
        dim, train = log(32, 1024), rng.random() < 0.7
        n = log(1, min(131072, 65536 * 8 * 768 // (slots * max(entries, 1) * dim)))
        return {"kind": kind, "n": n, "slots": slots, "entries": entries, "dim": dim,
                "dtype": rng.choice(("bf16", "bf16", "fp16", "fp32")), "train": train,
                "learned": train and entries > 0 and rng.random() < 0.3}
    page = rng.choice((16, 32, 64, 128, 256))
    dim = rng.choice((64, 64, 80, 96, 128, 128, 192, 256))
    dtype = rng.choice(("bf16", "bf16", "fp16"))
    codes = rng.choice(("int8", "int8", "fp8", "fp8", dtype))
    heads = rng.choice((1, 2, 3, 4, 5, 8, 8, 12, 16))
    if kind == "cache":
        write = log(1, 16384)
        read = rng.choice((0, write, log(write, 32768)))
        return {"kind": kind, "write": write, "read": read, "heads": heads, "dim": dim, "page": page, "codes": codes,
                "dtype": dtype, "skip": rng.random() < 0.5}
    seqs, group = log(1, 64), rng.choice((1, 2, 3, 4, 4, 8))
    width = rng.choice((1, log(2, 64), log(2, 64)))
    context = log(1, min(131072, 64 * 8192 * 8 * 128 // (seqs * heads * dim)))
    while seqs * heads * group * width * context > 2 * 32 * 64 * 131072:  # no drawn case costs more than the largest
        context = context // 2
    return {"kind": kind, "seqs": seqs, "width": width, "heads": heads, "group": group, "dim": dim, "page": page,
            "codes": codes, "dtype": dtype, "context": context, "ragged": rng.random() < 0.7,
            "lse": rng.random() < 0.5}


# ---------------------------------------------------------------------------------------------------------- inputs


def _lengths(case):
    """The sequences' cached lengths and tree widths: from the case alone. Ragged: down to a quarter of the context; where
    there are three sequences or more, the first has no context."""
    B, T, C = case["seqs"], case["width"], case["context"]
    if not case["ragged"]:
        return [C] * B, [T] * B
    lengths = [C - (b * 7919) % (3 * C // 4 + 1) for b in range(B)]
    widths = [T - (b * 5) % (T // 2 + 1) for b in range(B)]
    if B >= 3:
        lengths[0] = 0
    return lengths, widths


def _padded(dim):
    return (dim + 63) // 64 * 64


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _quantised(x, codes):
    """x [..., dim] as its codes and scales (the plain form, 32 bits)."""
    x = x.float()
    if codes in ("bf16", "fp16"):
        return x.to(CODES[codes]), None
    a = x.abs().amax(-1)
    top = torch.full_like(a, TOP[codes])  # a tensor: dividing by or into a number is a product with a reciprocal
    y = x * torch.where(a > 0, top / a, 0.0)[..., None]
    return (y.round() if codes == "int8" else y).to(CODES[codes]), a / top


def _stored(heads, pages, page, dim, codes, g):
    """A filled cache: codes and scales of random rows."""
    x = torch.randn((pages, heads, page, dim), generator=g, device="cuda")
    c, s = _quantised(x, codes)
    del x
    if _padded(dim) != dim:
        full = torch.zeros((pages, heads, page, _padded(dim)), dtype=c.dtype, device="cuda")
        _bits(full)[..., :dim] = _bits(c)
        c = full
    return c, s


def _bits(t):
    """The codes as integers of their size: elementary indexing has no 8-bit floats."""
    return t.view({1: torch.uint8, 2: torch.int16}[t.element_size()])


def _framework(module):
    if PACKAGE not in sys.path:
        sys.path.insert(0, PACKAGE)
    import importlib

    return importlib.import_module("ngram_amd." + module)


def prepare(case, seed):
    return {"embed": _prepare_embed, "cache": _prepare_cache, "tree": _prepare_tree}[case["kind"]](case, seed)


def _prepare_embed(case, seed):
    """Tokens are Zipf(1.1) over permuted ids; half the slots hold a row, each of 1 to `entries` candidates whose weights
    are descending counts' shares in units of 1 / 65535, zeros behind them, as a hint directory holds them."""
    g = _generator(seed)
    n, S, E, D = case["n"], case["slots"], case["entries"], case["dim"]
    dt = DTYPES[case["dtype"]]
    s = SimpleNamespace(kind="embed", train=case["train"], learned=case["learned"], scale=math.sqrt(D) if E == 0 else 0.5)
    s.table = (torch.randn((VOCAB, D), generator=g, device="cuda") * 0.05).to(dt)
    cdf = (torch.arange(1, VOCAB + 1, device="cuda", dtype=torch.float64) ** -1.1).cumsum(0)
    u = torch.rand(n * S * max(E, 1), generator=g, device="cuda", dtype=torch.float64) * cdf[-1]
    ranks = torch.searchsorted(cdf, u).clamp_(max=VOCAB - 1)
    tokens = torch.randperm(VOCAB, generator=g, device="cuda")[ranks]
    s.weights = s.cell = None
    if E == 0:
        s.tokens = tokens.reshape(n)
    else:
        lead = (n,) if S == 1 else (n, S)
        s.tokens = tokens.reshape(*lead, E)
        hinted = torch.rand(lead, generator=g, device="cuda") < 0.5
        s.cell = torch.where(hinted, torch.randint(1, 336, lead, generator=g, device="cuda"), 0)
        used = torch.arange(E, device="cuda") < torch.randint(1, E + 1, (*lead, 1), generator=g, device="cuda")
        counts = torch.randint(1, 1000, (*lead, E), generator=g, device="cuda").sort(-1, descending=True).values * used
        share = counts.float() / counts.sum(-1, keepdim=True).float()
        s.weights = (share * 65535).round() / 65535 * hinted[..., None]
    if s.train:
        s.grad = torch.randn((n, D), generator=g, device="cuda").to(dt)
        s.table.requires_grad_(True)
        if s.learned:
            s.weights.requires_grad_(True)
    if own:
        s.embed = _framework("embed").embed
    return s


def _prepare_cache(case, seed):
    """A cache that holds the sequence read, its pages in a random order; the tokens written are the sequence's last."""
    g = _generator(seed)
    W, R, H, D, P = case["write"], case["read"], case["heads"], case["dim"], case["page"]
    n = max(W, R)
    pages = -(-n // P) + 3
    s = SimpleNamespace(kind="cache", read=R, page=P, dim=D, codes=case["codes"], dtype=DTYPES[case["dtype"]],
                        skip=case["skip"])
    s.k, s.k_scale = _stored(H, pages, P, D, s.codes, g)
    s.v, s.v_scale = _stored(H, pages, P, D, s.codes, g)
    order = torch.randperm(pages, generator=g, device="cuda")
    at = torch.arange(n, device="cuda")
    slots = order[at // P] * P + at % P
    if case["skip"]:
        slots = torch.where(torch.rand(n, generator=g, device="cuda") < 0.1, -1, slots)
    s.slots, s.new = slots, slots[n - W:]
    s.new_k = torch.randn((W, H, D), generator=g, device="cuda").to(s.dtype)
    s.new_v = torch.randn((W, H, D), generator=g, device="cuda").to(s.dtype)
    if own:
        s.cache = _framework("kvcache").KVCache(s.k, s.v, s.k_scale, s.v_scale, dim=D)
    return s


def _prepare_tree(case, seed):
    """Trees of random shape (a token's parent is any earlier one, or the context), page tables over pages in a random
    order whose unused entries are -1, queries of twice the keys' size (so that the softmax is not flat)."""
    g = _generator(seed)
    B, T, H, G, D, P = (case[k] for k in ("seqs", "width", "heads", "group", "dim", "page"))
    lengths, widths = _lengths(case)
    s = SimpleNamespace(kind="tree", dim=D, heads=H, page=P, lse=case["lse"], scale=1 / math.sqrt(D),
                        dtype=DTYPES[case["dtype"]], longest=max(lengths) + T)
    used = [-(-(n + T) // P) for n in lengths]
    pages = sum(used) + 2
    order = torch.randperm(pages, generator=g, device="cuda").int().cpu()
    table = torch.full((B, max(used)), -1, dtype=torch.int32)
    at = 0
    for b, m in enumerate(used):
        table[b, :m] = order[at:at + m]
        at += m
    parents = (torch.rand((B, T), generator=g, device="cuda") * (torch.arange(T, device="cuda") + 1)).long().cpu() - 1
    mask = torch.zeros((B, T), dtype=torch.int64)
    for i in range(T):
        above = torch.where(parents[:, i] >= 0, mask[torch.arange(B), parents[:, i].clamp(min=0)], 0)
        mask[:, i] = above | (1 << i if i < 63 else -(1 << 63))
    s.table, s.mask = table.cuda(), mask.cuda() if T > 1 else None
    s.lengths = torch.tensor(lengths, dtype=torch.int32).cuda()
    s.widths = torch.tensor(widths, dtype=torch.int32).cuda() if case["ragged"] else None
    s.k, s.k_scale = _stored(H, pages, P, D, case["codes"], g)
    s.v, s.v_scale = _stored(H, pages, P, D, case["codes"], g)
    s.q = (torch.randn((B, T, H * G, D), generator=g, device="cuda") * 2).to(s.dtype)
    if own:
        s.cache = _framework("kvcache").KVCache(s.k, s.v, s.k_scale, s.v_scale, dim=D)
        s.attend = _framework("tree").tree_attention
    return s


# ------------------------------------------------------------------------------------------------------------- run


def run(state):
    return {"embed": _run_embed, "cache": _run_cache, "tree": _run_tree}[state.kind](state)


def _run_embed(s):
    if not own:
        return _plain_embed(s)
    out = s.embed(s.table, s.tokens, s.weights, s.cell, scale=s.scale)
    if not s.train:
        return out
    wanted = [s.table, s.weights] if s.learned else [s.table]
    return [out, *torch.autograd.grad(out, wanted, s.grad)]


def _plain_embed(s):
    table, n, D = s.table.detach(), s.tokens.shape[0], s.table.shape[1]
    flat = s.tokens.reshape(n, -1)
    rows = table[flat].float()  # [n, m, D]
    if s.weights is None:
        has = w = torch.ones(flat.shape, device=rows.device)
    else:
        has = (s.cell > 0)[..., None].expand(s.weights.shape).reshape(n, -1).float()
        w = s.weights.detach().reshape(n, -1) * has
    out = (torch.matmul(w[:, None, :], rows)[:, 0] * s.scale).to(table.dtype)
    if not s.train:
        return out
    up = s.grad.float() * s.scale
    grad = torch.zeros((VOCAB, D), device=rows.device)
    grad.index_add_(0, flat.reshape(-1), (w[..., None] * up[:, None, :]).reshape(-1, D))
    if not s.learned:
        return [out, grad.to(table.dtype)]
    return [out, grad.to(table.dtype), ((rows * up[:, None, :]).sum(-1) * has).reshape(s.weights.shape)]


def _run_cache(s):
    if own:
        s.cache.write(s.new_k, s.new_v, s.new)
        if s.read:
            return list(s.cache.read(s.slots, dtype=s.dtype))
    else:
        for_k = _plain_write(s, s.k, s.k_scale, s.new_k)
        for_v = _plain_write(s, s.v, s.v_scale, s.new_v)
        if s.read:
            return [_plain_read(s, *for_k), _plain_read(s, *for_v)]
    return [s.k, s.v] if s.k_scale is None else [s.k, s.v, s.k_scale, s.v_scale]


def _plain_write(s, held, scales, x):
    codes, scale = _quantised(x, s.codes)
    at = s.new >= 0 if s.skip else slice(None)
    page, row = s.new[at] // s.page, s.new[at] % s.page
    heads = torch.arange(held.shape[1], device=held.device)
    _bits(held)[..., :s.dim][page[:, None], heads, row[:, None]] = _bits(codes)[at]
    if scales is not None:
        scales[page[:, None], heads, row[:, None]] = scale[at]
    return held, scales


def _plain_read(s, held, scales):
    at = s.slots.clamp(min=0)
    page, row = at // s.page, at % s.page
    heads = torch.arange(held.shape[1], device=held.device)
    x = _bits(held)[page[:, None], heads, row[:, None]].view(held.dtype)[..., :s.dim].float()
    if scales is not None:
        x = x * scales[page[:, None], heads, row[:, None]][..., None]
    return torch.where((s.slots >= 0)[:, None, None], x, 0.0).to(s.dtype)


def _run_tree(s):
    if own:
        return s.attend(s.q, s.cache, s.table, s.lengths, s.mask, s.widths, scale=s.scale, return_lse=s.lse)
    B, T, Hq, D = s.q.shape
    at = s.table.clamp(min=0).long()
    k, v = _plain_dense(s, s.k, s.k_scale, at), _plain_dense(s, s.v, s.v_scale, at)  # [B, H, L, D]
    L = k.shape[2]
    q = s.q.float().reshape(B, T, s.heads, -1, D).permute(0, 2, 3, 1, 4).reshape(B, s.heads, -1, D)  # [B, H, G * T, D]
    score = torch.matmul(q, k.transpose(2, 3).contiguous()) * s.scale
    del k
    place = torch.arange(L, device=q.device) - s.lengths[:, None]  # [B, L]: the place in the tree, negative before it
    row = torch.arange(T, device=q.device)
    tree = place.clamp(0, 63)[:, None, :]
    seen = place[:, None, :] <= row[:, None] if s.mask is None else (s.mask[:, :, None] >> tree) & 1 > 0
    width = torch.full_like(s.lengths, T) if s.widths is None else s.widths
    seen = (place[:, None, :] < 0) | (seen & (place < width[:, None])[:, None, :])
    seen = seen & (row < width[:, None])[:, :, None]  # [B, T, L]
    score = score.view(B, s.heads, -1, T, L).masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    p = score.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(B, s.heads, -1, L), v).view(B, s.heads, -1, T, D)
    out = torch.where(total > 0, out / total, 0.0).permute(0, 3, 1, 2, 4).reshape(B, T, Hq, D).to(s.dtype)
    if not s.lse:
        return out
    return [out, (total.log() + top)[..., 0].permute(0, 3, 1, 2).reshape(B, T, Hq)]


def _plain_dense(s, held, scales, at):
    x = _bits(held)[at].view(held.dtype)[..., :s.dim].float()  # [B, pages, H, page, D]
    if scales is not None:
        x = x * scales[at][..., None]
    B, m, H, P, D = x.shape
    return x.transpose(1, 2).reshape(B, H, m * P, D)[:, :, :s.longest].contiguous()


# ------------------------------------------------------------------------------------------------------------ work


def work(case):
    if case["kind"] == "embed":
        n, S, E, D = case["n"], case["slots"], case["entries"], case["dim"]
        size = 4 if case["dtype"] == "fp32" else 2
        m = n * S * max(E, 1)
        used = m if E == 0 else m * (E + 1) / (4 * E)  # half the slots, of 1 to E candidates
        rows = min(VOCAB, used)
        index = 8 * m + (0 if E == 0 else 4 * m + 8 * n * S)
        bytes_, flops = index + (rows + n) * D * size, 2 * used * D
        if case["train"]:
            bytes_ += (n + VOCAB) * D * size + (4 * m if case["learned"] else 0)
            flops += 2 * used * D + (m * D if case["learned"] else 0)
        return {"bytes": bytes_, "flops": flops}
    H, D = case["heads"], case["dim"]
    code = 2 if case["codes"] in ("bf16", "fp16") else 1
    held = 2 * H * (D * code + (4 if code == 1 else 0))  # a token's keys and values
    if case["kind"] == "cache":
        rows = 2 * H * D * 2
        n = case["write"] + case["read"]
        return {"bytes": n * (held + rows) + 8 * n, "flops": 3.0 * n * H * D}
    lengths, widths = _lengths(case)
    G, T = case["group"], case["width"]
    tokens = sum(lengths) + sum(widths)
    rows = 2 * case["seqs"] * T * H * G * D * 2
    seen = sum(w * n for n, w in zip(lengths, widths)) + sum(w * (w + 1) / 2 for w in widths)
    return {"bytes": tokens * held + rows + (4 * case["seqs"] * T * H * G if case["lse"] else 0),
            "flops": 4.0 * H * G * D * seen}


# ----------------------------------------------------------------------------------------------------------- exact


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    return {"embed": _exact_embed, "cache": _exact_cache, "tree": _exact_tree}[case["kind"]](s)


def _exact_embed(s):
    table = s.table.detach().double()
    n, D = s.tokens.shape[0], table.shape[1]
    tokens = s.tokens.reshape(n, -1)
    weights = torch.ones(tokens.shape, device="cuda", dtype=torch.float64)
    counted = torch.ones(tokens.shape, device="cuda", dtype=torch.bool)
    if s.weights is not None:
        weights = s.weights.detach().double().reshape(n, -1)
        counted = (s.cell > 0).reshape(n, -1).repeat_interleave(s.weights.shape[-1], 1)
    out = torch.zeros((n, D), device="cuda", dtype=torch.float64)
    grad = torch.zeros((VOCAB, D), device="cuda", dtype=torch.float64)
    slopes = torch.zeros(tokens.shape, device="cuda", dtype=torch.float64)
    up = s.grad.double() if s.train else None
    for e in range(tokens.shape[1]):  # one entry of every position at a time
        take = counted[:, e].nonzero()[:, 0]
        t, w = tokens[take, e], weights[take, e, None] * s.scale
        out[take] += w * table[t]
        if s.train:
            grad.index_put_((t,), w * up[take], accumulate=True)
            slopes[take, e] = s.scale * (table[t] * up[take]).sum(1)
    if not s.train:
        return out
    return [out, grad, slopes.reshape(s.weights.shape)] if s.learned else [out, grad]


def _exact_codes(x, codes):
    """The codes as the values they stand for before the scale, and the scales."""
    x = x.double()
    if codes in ("bf16", "fp16"):
        return x, None
    a = x.abs().max(-1, keepdim=True).values
    y = torch.where(a > 0, x / torch.where(a > 0, a, 1.0) * TOP[codes], 0.0)
    if codes == "int8":
        return torch.round(y), a / TOP[codes]
    e = torch.frexp(y.abs()).exponent.double() - 1  # e4m3: steps of 2^(e - 3), no finer than 2^-9
    step = torch.exp2(e.clamp(min=-6) - 3)
    return torch.round(y / step) * step, a / TOP[codes]


def _exact_cache(s):
    whole = []
    for held, scales, new in ((s.k, s.k_scale, s.new_k), (s.v, s.v_scale, s.new_v)):
        pages, H, P, DP = held.shape
        c = held.float().double().permute(0, 2, 1, 3).reshape(pages * P, H, DP)
        z = None if scales is None else scales.double().permute(0, 2, 1).reshape(pages * P, H, 1).clone()
        codes, scale = _exact_codes(new, s.codes)
        for_slot = s.new[s.new >= 0]
        c[for_slot, :, :s.dim] = codes[s.new >= 0]
        if z is not None:
            z[for_slot] = scale[s.new >= 0]
        if s.read:
            x = c[s.slots.clamp(min=0), :, :s.dim]
            x = x if z is None else x * z[s.slots.clamp(min=0)]
            x[s.slots < 0] = 0
            whole.append(x)
        else:
            values = None if s.codes == "int8" else c.reshape(pages, P, H, DP).permute(0, 2, 1, 3).contiguous()
            whole.append((values, None if z is None else z.reshape(pages, P, H).permute(0, 2, 1).contiguous()))
    if s.read:
        return whole
    (k, k_scale), (v, v_scale) = whole
    return [k, v] if k_scale is None else [k, v, k_scale, v_scale]


def _exact_tree(s):
    B, T, Hq, D = s.q.shape
    G = Hq // s.heads
    out = torch.zeros((B, T, Hq, D), device="cuda", dtype=torch.float64)
    lse = torch.full((B, T, Hq), -math.inf, device="cuda", dtype=torch.float64)
    lengths = s.lengths.tolist()
    widths = [T] * B if s.widths is None else s.widths.tolist()
    masks = [[(1 << (i + 1)) - 1 for i in range(T)]] * B if s.mask is None else s.mask.tolist()
    for b in range(B):
        n, w = lengths[b], widths[b]
        if n + w == 0:
            continue
        sees = torch.ones((w, n + w), dtype=torch.bool)
        for i in range(w):
            for j in range(w):
                sees[i, n + j] = bool(masks[b][i] >> j & 1)
        sees = sees.cuda()
        pages = s.table[b, :-(-(n + w) // s.page)].long()
        for h in range(s.heads):
            k, v = (held[pages, h].float().double().reshape(-1, held.shape[3])[:n + w, :D] for held in (s.k, s.v))
            if s.k_scale is not None:
                k = k * s.k_scale[pages, h].double().reshape(-1, 1)[:n + w]
                v = v * s.v_scale[pages, h].double().reshape(-1, 1)[:n + w]
            for r in range(h * G, (h + 1) * G):
                a = (s.q[b, :w, r].double() @ k.T) * s.scale
                a[~sees] = -math.inf
                z = torch.logsumexp(a, 1)
                lse[b, :w, r] = z
                p = torch.exp(a - torch.where(z > -math.inf, z, 0.0)[:, None])
                out[b, :w, r] = p @ v
    return [out, lse] if s.lse else out
