"""The operators of a serving step over a paged q8 key/value cache, as measured
workloads: what a server does between the products of a decoder layer, and
after its last one.

A server keeps one pool of pages for all its sequences. Each step it appends
the new tokens' keys and values (queries and keys normalized per head and
rotated on the way), attends from the new tokens over the pages, and draws the
next tokens from the logits; when a sequence branches or the pool is tidied it
copies pages. The cases are those calls over the sizes that a server meets, in
their plain form (elementary tensor operations) and, with `own` set, through
this package's entry points. Head layouts are those of this repository's
decoder configurations and tests; weights and inputs are synthetic, made from
the seed.
"""
import math

import numpy as np
import torch

own = False

DEVICE = "cuda"
GROUP = 64
EPS = 1e-6
THETA = 1e6
VOCAB = 151936
LAYERS = 28
NO_PAGE = -1  # 0xffffffff as the tables' 32-bit words

# heads, kv_heads, head_dim: the 0.6B and 1.7B decoders, then other shapes.
HEADS = [(16, 8, 128), (16, 8, 128), (16, 8, 128), (8, 2, 64), (14, 2, 64), (12, 4, 128), (8, 1, 128), (4, 2, 256), (6, 2, 192)]


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------
def listed():
    q = {"heads": 16, "kv_heads": 8, "head_dim": 128}
    return [
        # One transcription's step after a 30 s prompt: the smallest call,
        # where launches and round trips count.
        {"name": "attend_step_b1", "kind": "attend", **q, "batch": 1, "tokens": 1, "first": 430, "ragged": False,
         "page_size": 16, "holes": 0},
        # A server's step for 16 sequences at 4096 positions: a stream of the cache.
        {"name": "attend_step_b16", "kind": "attend", **q, "batch": 16, "tokens": 1, "first": 4095, "ragged": False,
         "page_size": 16, "holes": 0},
        # A larger server's step, every sequence of another length.
        {"name": "attend_step_b61_ragged", "kind": "attend", **q, "batch": 61, "tokens": 1, "first": 5003, "ragged": True,
         "page_size": 64, "holes": 0},
        # The prompt of a 30 s clip, nothing cached before it.
        {"name": "attend_prompt_402", "kind": "attend", **q, "batch": 1, "tokens": 402, "first": 0, "ragged": False,
         "page_size": 16, "holes": 0},
        # The largest: a chunk of 512 tokens at the end of a long context.
        {"name": "attend_chunk_512_at_7680", "kind": "attend", **q, "batch": 1, "tokens": 512, "first": 7680,
         "ragged": False, "page_size": 32, "holes": 0},
        # A mixed step: steps and chunks together, pages of an odd size, pages
        # dropped from the middle, another head layout.
        {"name": "attend_mixed_b7", "kind": "attend", "heads": 14, "kv_heads": 2, "head_dim": 64, "batch": 7, "tokens": 133,
         "first": 2011, "ragged": True, "page_size": 24, "holes": 3},
        # The append of a server's step: one new token for each of 16 sequences.
        {"name": "append_step_b16", "kind": "append", **q, "batch": 16, "tokens": 1, "first": 4095, "ragged": False,
         "page_size": 16, "holes": 0},
        # The append of ragged prompts, three minutes of audio in all.
        {"name": "append_prompts_b5", "kind": "append", **q, "batch": 5, "tokens": 777, "first": 301, "ragged": True,
         "page_size": 48, "holes": 0},
        # A sequence forks into four: its last, half-filled page in every layer.
        {"name": "copy_fork_4", "kind": "copy", "kv_heads": 8, "head_dim": 128, "layers": LAYERS, "page_size": 16,
         "pages": 64, "pairs": 4, "fan": 4},
        # Compaction: the used pages behind a hole move to the front.
        {"name": "copy_compact_300", "kind": "copy", "kv_heads": 8, "head_dim": 128, "layers": LAYERS, "page_size": 16,
         "pages": 700, "pairs": 300, "fan": 1},
        # One sequence's next token.
        {"name": "sample_b1", "kind": "sample", "rows": 1, "count": VOCAB, "rule": "all"},
        # A server's rows, each with its own request's parameters.
        {"name": "sample_b64_mixed", "kind": "sample", "rows": 64, "count": VOCAB, "rule": "mixed"},
    ]


def log_int(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "append", "copy", "sample"])
    heads, kv_heads, head_dim = rng.choice(HEADS)
    page_size = rng.choice([16, 16, 32, 64, log_int(rng, 1, 128)])
    if kind == "attend":
        case = {"kind": kind, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "page_size": page_size,
                "ragged": rng.random() < 0.5, "holes": rng.choice([0, 0, 0, 2])}
        if rng.random() < 0.5:  # a server's step, perhaps with a few drafted tokens to check
            case.update(batch=log_int(rng, 1, 48), tokens=rng.choice([1, 1, 1, log_int(rng, 2, 16)]),
                        first=log_int(rng, 1, 4096))
        else:  # chunks
            case.update(batch=log_int(rng, 1, 4), tokens=log_int(rng, 17, 512),
                        first=rng.choice([0, log_int(rng, 1, 1500)]))
        return case
    if kind == "append":
        batch = log_int(rng, 1, 32)
        return {"kind": kind, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "batch": batch,
                "tokens": log_int(rng, 1, max(1, 2048 // batch)), "first": log_int(rng, 1, 4096),
                "ragged": rng.random() < 0.5, "page_size": page_size, "holes": rng.choice([0, 0, 2])}
    if kind == "copy":
        fan = rng.choice([1, 1, 2, 4, 8])
        page_size = log_int(rng, 1, 64)
        pairs = fan * log_int(rng, 1, max(1, 4000 // (page_size * fan)))
        return {"kind": kind, "kv_heads": kv_heads, "head_dim": head_dim, "layers": rng.choice([1, LAYERS, log_int(rng, 1, LAYERS)]),
                "page_size": page_size, "pages": pairs + pairs // fan + log_int(rng, 1, 40), "pairs": pairs, "fan": fan}
    return {"kind": kind, "rows": log_int(rng, 1, 64), "count": rng.choice([VOCAB, VOCAB, log_int(rng, 1000, VOCAB)]),
            "rule": rng.choice(["all", "mixed", "top_k", "top_p", "min_p", "free", "greedy"])}


# ---------------------------------------------------------------------------
# What the case alone decides: the sequences' lengths
# ---------------------------------------------------------------------------
def lengths(case):
    """(new tokens, positions cached before them) of each sequence."""
    new, first = [], []
    for b in range(case["batch"]):
        if case["ragged"]:
            new.append(1 + (case["tokens"] - 1) * ((7 * b + 10) % 11) // 10)
            first.append(case["first"] * ((5 * b + 13) % 17) // 16)
        else:
            new.append(case["tokens"])
            first.append(case["first"])
    return new, first


def padding(case):
    """Rows of the buffers behind the last sequence's: a server pads its row
    buffers. A step of one token each has none."""
    return 3 if case["ragged"] and case["tokens"] > 1 else 0


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
class Inputs:
    """Values in a fixed order from one seed."""

    def __init__(self, seed):
        self.generator = torch.Generator(device=DEVICE)
        self.generator.manual_seed(1000003 * int(seed) + 29)

    def normal(self, *shape):
        return torch.randn(*shape, generator=self.generator, device=DEVICE, dtype=torch.float32)

    def uniform(self, *shape):
        return torch.rand(*shape, generator=self.generator, device=DEVICE, dtype=torch.float32)

    def permutation(self, n):
        return torch.randperm(n, generator=self.generator, device=DEVICE)

    def codes(self, rows, width):
        """Stored codes of rows of about normal values: the largest of 64 is
        near 128 steps, so a standard deviation is near 50."""
        out = torch.empty(rows, width, device=DEVICE, dtype=torch.uint8)
        step = max(1, (1 << 26) // width)
        for r in range(0, rows, step):
            n = min(step, rows - r)
            out[r:r + n] = (self.normal(n, width) * 50.0).round_().clamp_(-128, 127).add_(128).to(torch.uint8)
        return out

    def scales(self, rows, groups):
        return (0.014 + 0.012 * self.uniform(rows, groups)).half()


class State:
    """What a server holds between calls."""

    def __init__(self, case):
        self.case = case
        self.cache = None


_context = None


def context():
    """The program's one context: a device and a stream."""
    global _context
    if _context is None:
        import qwenscriber_amd as qa

        _context = qa.Context(0)
    return _context


def pool(s, i, layers, pages, page_size, kv_heads, head_dim):
    """One pool of pages: codes and scales of keys and values."""
    width = kv_heads * head_dim
    s.layers, s.pages, s.page_size, s.kv_heads, s.head_dim = layers, pages, page_size, kv_heads, head_dim
    rows = layers * pages * page_size
    s.k_codes, s.k_scales = i.codes(rows, width), i.scales(rows, width // GROUP)
    s.v_codes, s.v_scales = i.codes(rows, width), i.scales(rows, width // GROUP)


def sequences(s, i, case):
    """The batch of sequences: rows, lengths and page tables."""
    new, first = lengths(case)
    size = case["page_size"]
    need = [-(-(f + n) // size) for n, f in zip(new, first)]
    s.new, s.first, s.table_pages = new, first, max(need) + 1
    s.total, s.rows = sum(new), sum(new) + padding(case)
    pages = sum(need) + 5
    order = i.permutation(pages).to(torch.int32)
    tables = torch.full((case["batch"], s.table_pages), NO_PAGE, device=DEVICE, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        tables[b, :n] = order[at:at + n]
        at += n
        # Pages dropped from the middle of a long sequence, its first kept.
        if case["holes"] and n > case["holes"] + 4:
            tables[b, 2:2 + case["holes"]] = NO_PAGE
    s.tables = tables
    starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    s.starts = torch.from_numpy(starts).to(DEVICE)
    s.first_dev = torch.tensor(first, device=DEVICE, dtype=torch.int32)
    # Each row's sequence and position, and where a (sequence, token) row is
    # (the last, spare row for tokens that a shorter sequence has not).
    seq = np.repeat(np.arange(case["batch"]), new)
    within = np.arange(s.total) - starts[seq]
    s.row_seq = torch.from_numpy(seq).to(DEVICE)
    s.row_pos = torch.from_numpy(np.asarray(first)[seq] + within).to(DEVICE)
    # The rows whose position has a page.
    s.kept = torch.nonzero(tables[s.row_seq, s.row_pos // size] != NO_PAGE)[:, 0]
    t = np.arange(max(new))[None, :]
    s.row_at = torch.from_numpy(np.where(t < np.asarray(new)[:, None], starts[:-1, None] + t, s.rows)).to(DEVICE)
    return pages


# ---------------------------------------------------------------------------
# Attention of new tokens over the pages
# ---------------------------------------------------------------------------
def prepare_attend(case, seed):
    s, i = State(case), Inputs(seed)
    pages = sequences(s, i, case)
    pool(s, i, 1, pages, case["page_size"], case["kv_heads"], case["head_dim"])
    s.heads = case["heads"]
    width = s.heads * s.head_dim
    # A trained model's scores spread over a few units.
    s.query = 2.0 * i.normal(s.rows, width)
    s.out = torch.zeros(s.rows, width, device=DEVICE)
    return s


def stored(codes, scales, rows, dtype):
    """The values that stored rows stand for."""
    c = codes[rows].to(dtype) - 128
    return (c.unflatten(-1, (-1, GROUP)) * scales[rows].to(dtype).unsqueeze(-1)).flatten(-2)


def attend_plain(s):
    """Every sequence's context gathered to the longest one's length, then
    scores, weights and the weighted sum, position by mask."""
    batch, heads, kv_heads, dim = s.case["batch"], s.heads, s.kv_heads, s.head_dim
    tokens, ratio = max(s.new), heads // kv_heads
    positions = torch.arange(max(n + f for n, f in zip(s.new, s.first)), device=DEVICE)
    page = s.tables[:, positions // s.page_size].long()
    there = (page >= 0) & (page < s.pages)
    rows = torch.where(there, page * s.page_size + positions % s.page_size, 0)
    keys = stored(s.k_codes, s.k_scales, rows, torch.float32).unflatten(-1, (kv_heads, dim))
    values = stored(s.v_codes, s.v_scales, rows, torch.float32).unflatten(-1, (kv_heads, dim))
    keys, values = keys.permute(0, 2, 3, 1).contiguous(), values.permute(0, 2, 1, 3).contiguous()
    padded = torch.cat([s.query, torch.zeros_like(s.query[:1])])[s.row_at]
    q = padded.unflatten(-1, (kv_heads, ratio, dim)).permute(0, 2, 3, 1, 4).reshape(batch, kv_heads, ratio * tokens, dim)
    scores = torch.matmul(q, keys) / math.sqrt(dim)
    last = s.first_dev.long()[:, None] + torch.arange(tokens, device=DEVICE)
    seen = there[:, None, :] & (positions <= last[:, :, None])
    scores = scores.unflatten(2, (ratio, tokens)).masked_fill(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    weights = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = weights.sum(-1, keepdim=True)
    got = torch.matmul(weights.flatten(2, 3), values).unflatten(2, (ratio, tokens))
    got = torch.where(total > 0, got / total, 0.0)
    got = got.permute(0, 3, 1, 2, 4).reshape(batch * tokens, heads * dim)
    out = torch.zeros(s.rows + 1, heads * dim, device=DEVICE)
    out[s.row_at.reshape(-1)] = got
    return out[:s.rows]


def paged(s):
    """This package's descriptors of the pool and of the batch."""
    import qwenscriber_amd as qa

    if s.cache is None:  # a server makes its pool's once
        s.cache = qa.PagedCache(s.layers, s.pages, s.page_size, s.kv_heads, s.head_dim, s.k_scales.data_ptr(),
                                s.k_codes.data_ptr(), s.v_scales.data_ptr(), s.v_codes.data_ptr())
    return s.cache, qa.PagedBatch(s.case["batch"], s.rows, s.table_pages,
                                  None if s.case["tokens"] == 1 else s.starts.data_ptr(), s.first_dev.data_ptr(),
                                  s.tables.data_ptr())


def attend_own(s):
    cache, batch = paged(s)
    context().paged_attention(cache, 0, batch, s.out.data_ptr(), s.query.data_ptr(), s.heads * s.head_dim, s.heads)
    return s.out


def exact_attend(case, seed):
    s = prepare_attend(case, seed)
    pairs = sum(n * (f + n) for n, f in zip(s.new, s.first))
    if pairs * s.heads * s.head_dim > 3e10:
        return None
    ratio, dim = s.heads // s.kv_heads, s.head_dim
    out = torch.zeros(s.rows, s.heads * dim, device=DEVICE, dtype=torch.float64)
    row = 0
    for b in range(case["batch"]):
        n, f = s.new[b], s.first[b]
        where = torch.arange(f + n, device=DEVICE)
        page = s.tables[b].long()[where // s.page_size]
        where, page = where[page != NO_PAGE], page[page != NO_PAGE]
        rows = page * s.page_size + where % s.page_size
        mask = where[None, :] > (f + torch.arange(n, device=DEVICE))[:, None]
        for g in range(s.kv_heads):
            cols = slice(g * dim, (g + 1) * dim)
            k, v = (((c[rows, cols].double() - 128).reshape(len(rows), -1, GROUP)
                     * z[rows, g * dim // GROUP:(g + 1) * dim // GROUP].double()[:, :, None]).reshape(len(rows), dim)
                    for c, z in ((s.k_codes, s.k_scales), (s.v_codes, s.v_scales)))
            for h in range(g * ratio, (g + 1) * ratio):
                at = slice(h * dim, (h + 1) * dim)
                score = s.query[row:row + n, at].double() @ k.t().contiguous() / math.sqrt(dim)
                weight = torch.softmax(score.masked_fill(mask, -math.inf), dim=1).nan_to_num(0.0)
                out[row:row + n, at] = weight @ v
        row += n
    return out


def row_bytes(case):
    """One position's stored rows: key and value codes and scales."""
    width = case["kv_heads"] * case["head_dim"]
    return 2 * (width + width // GROUP * 2)


def work_attend(case):
    new, first = lengths(case)
    width = case["heads"] * case["head_dim"]
    pairs = sum(n * f + n * (n + 1) // 2 for n, f in zip(new, first))
    return {"bytes": sum(n + f for n, f in zip(new, first)) * row_bytes(case) + 8 * sum(new) * width,
            "flops": 4 * pairs * width}


# ---------------------------------------------------------------------------
# Norms, rotation and the append
# ---------------------------------------------------------------------------
def prepare_append(case, seed):
    s, i = State(case), Inputs(seed)
    pages = sequences(s, i, case)
    pool(s, i, 1, pages, case["page_size"], case["kv_heads"], case["head_dim"])
    s.heads = case["heads"]
    dim = s.head_dim
    s.qkv = i.normal(s.rows, (s.heads + 2 * s.kv_heads) * dim)
    s.q_norm, s.k_norm = 1.0 + 0.3 * i.normal(dim), 1.0 + 0.3 * i.normal(dim)
    s.table_positions = s.table_pages * s.page_size
    angle = torch.arange(s.table_positions, device=DEVICE, dtype=torch.float64)[:, None] * THETA ** (
        -2.0 * torch.arange(dim // 2, device=DEVICE, dtype=torch.float64) / dim)
    s.cos, s.sin = torch.cos(angle).float(), torch.sin(angle).float()
    s.query = torch.zeros(s.rows, s.heads * dim, device=DEVICE)
    return s


def quantized(x):
    """The cache's q8 rows of f32 values: f16 scales and biased codes."""
    groups = x.unflatten(-1, (-1, GROUP))
    scale = (groups.abs().amax(-1) / 128).half()
    step = scale.float().unsqueeze(-1)
    ratio = torch.where(step == 0, 0.0, (groups.double() / step.double()).float())
    codes = torch.where(ratio >= 0, torch.floor(ratio + 0.5), torch.ceil(ratio - 0.5)).clamp(-128, 127)
    return (codes + 128).to(torch.uint8).flatten(-2), scale


def append_plain(s):
    """The rows in 64 bits up to the one rounding to f32: a stored code is a
    rounding of that value, and next to a border 32 bits lose it."""
    dim, heads, kv_heads, n = s.head_dim, s.heads, s.kv_heads, s.total
    x = s.qkv[:n].unflatten(-1, (heads + 2 * kv_heads, dim))
    qk, v = x[:, :heads + kv_heads].double(), x[:, heads + kv_heads:]
    weight = torch.cat([s.q_norm.expand(heads, dim), s.k_norm.expand(kv_heads, dim)]).double()
    y = qk / torch.sqrt((qk * qk).mean(-1, keepdim=True) + float(np.float32(EPS))) * weight
    cos, sin = s.cos[s.row_pos].double().unsqueeze(1), s.sin[s.row_pos].double().unsqueeze(1)
    low, high = y[..., :dim // 2], y[..., dim // 2:]
    y = torch.cat([low * cos - high * sin, high * cos + low * sin], -1).float()
    query = torch.zeros(s.rows, heads * dim, device=DEVICE)
    query[:n] = y[:, :heads].flatten(1)
    seq, pos = s.row_seq[s.kept], s.row_pos[s.kept]
    rows = s.tables[seq, pos // s.page_size].long() * s.page_size + pos % s.page_size
    planes = []
    for codes, scales, value in ((s.k_codes, s.k_scales, y[:, heads:]), (s.v_codes, s.v_scales, v)):
        c, z = quantized(value.flatten(1))
        planes += [codes.index_copy_(0, rows, c[s.kept]), scales.index_copy_(0, rows, z[s.kept])]
    return [query] + planes


def append_own(s):
    cache, batch = paged(s)
    dim = s.head_dim
    context().paged_append(cache, 0, batch, s.qkv.data_ptr(), (s.heads + 2 * s.kv_heads) * dim, s.heads,
                           s.q_norm.data_ptr(), s.k_norm.data_ptr(), EPS, s.cos.data_ptr(), s.sin.data_ptr(),
                           s.table_positions, s.query.data_ptr(), s.heads * dim)
    # The codes are bytes that the format defines to the last bit: compared
    # as they are, with their scales.
    return [s.query, s.k_codes, s.k_scales, s.v_codes, s.v_scales]


def exact_append(case, seed):
    s = prepare_append(case, seed)
    dim, heads, kv_heads = s.head_dim, s.heads, s.kv_heads
    query = torch.zeros(s.rows, heads * dim, device=DEVICE, dtype=torch.float64)
    k_scales, v_scales = s.k_scales.double(), s.v_scales.double()
    groups = kv_heads * dim // GROUP
    for b in range(case["batch"]):
        begin = int(s.starts[b])
        n, f = s.new[b], s.first[b]
        where = f + torch.arange(n, device=DEVICE)
        page = s.tables[b].long()[where // s.page_size]
        kept = page != NO_PAGE
        rows = (page * s.page_size + where % s.page_size)[kept]
        turn = torch.complex(s.cos[where].double(), s.sin[where].double())
        for h in range(heads + kv_heads):
            x = s.qkv[begin:begin + n, h * dim:(h + 1) * dim].double()
            x = x * (s.q_norm if h < heads else s.k_norm).double() * torch.rsqrt(x.square().sum(1, keepdim=True) / dim + float(np.float32(EPS)))
            z = torch.complex(x[:, :dim // 2], x[:, dim // 2:]) * turn
            x = torch.cat([z.real, z.imag], 1)
            if h < heads:
                query[begin:begin + n, h * dim:(h + 1) * dim] = x
            else:
                g = (h - heads) * dim // GROUP
                k_scales[rows, g:g + dim // GROUP] = x.reshape(n, -1, GROUP).abs().amax(2)[kept] / 128
        v = s.qkv[begin:begin + n, (heads + kv_heads) * dim:].double()
        v_scales[rows] = v.reshape(n, groups, GROUP).abs().amax(2)[kept] / 128
    return [query, None, k_scales, None, v_scales]


def work_append(case):
    new, _ = lengths(case)
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["head_dim"]
    per_row = 4 * (2 * heads + 2 * kv_heads) * dim + row_bytes(case)
    return {"bytes": sum(new) * (per_row + 4 * dim), "flops": sum(new) * 10 * (heads + kv_heads) * dim}


# ---------------------------------------------------------------------------
# Copies of pages
# ---------------------------------------------------------------------------
def prepare_copy(case, seed):
    s, i = State(case), Inputs(seed)
    pool(s, i, case["layers"], case["pages"], case["page_size"], case["kv_heads"], case["head_dim"])
    shape = (case["layers"], case["pages"], case["page_size"], -1)
    s.k_codes, s.k_scales = s.k_codes.view(shape), s.k_scales.view(shape)
    s.v_codes, s.v_scales = s.v_codes.view(shape), s.v_scales.view(shape)
    # `fan` copies of each source page.
    order = i.permutation(case["pages"])
    sources = case["pairs"] // case["fan"]
    s.src = order[:sources].repeat_interleave(case["fan"])
    s.dst = order[sources:sources + len(s.src)]
    # The host's allocator knows the pages it moves.
    s.src_host, s.dst_host = s.src.cpu().numpy().astype(np.uint32), s.dst.cpu().numpy().astype(np.uint32)
    return s


def copy_plain(s):
    for plane in (s.k_codes, s.k_scales, s.v_codes, s.v_scales):
        plane[:, s.dst] = plane[:, s.src]
    return [s.k_codes, s.k_scales, s.v_codes, s.v_scales]


def copy_own(s):
    cache, _ = paged_pool(s)
    context().paged_copy(cache, s.src_host, s.dst_host)
    return [s.k_codes, s.k_scales, s.v_codes, s.v_scales]


def paged_pool(s):
    import qwenscriber_amd as qa

    if s.cache is None:
        s.cache = qa.PagedCache(s.layers, s.pages, s.page_size, s.kv_heads, s.head_dim, s.k_scales.data_ptr(),
                                s.k_codes.data_ptr(), s.v_scales.data_ptr(), s.v_codes.data_ptr())
    return s.cache, None


def exact_copy(case, seed):
    s = prepare_copy(case, seed)
    out = []
    for plane in (s.k_codes, s.k_scales, s.v_codes, s.v_scales):
        new = plane.clone()
        for a, b in zip(s.src_host.tolist(), s.dst_host.tolist()):
            new[:, b] = plane[:, a]
        out.append(new.double() if new.dtype == torch.float16 else new)
    return out


def work_copy(case):
    pages = case["pairs"] + case["pairs"] // case["fan"]
    return {"bytes": pages * case["layers"] * case["page_size"] * row_bytes(case), "flops": 0}


# ---------------------------------------------------------------------------
# Sampling
# ---------------------------------------------------------------------------
# temperature, top_k (0: off), top_p (1: off), min_p (0: off)
RULES = {"all": [(0.8, 50, 0.95, 0.02)], "top_k": [(0.7, 20, 1.0, 0.0)], "top_p": [(1.0, 0, 0.9, 0.0)],
         "min_p": [(1.3, 0, 1.0, 0.05)], "free": [(1.0, 0, 1.0, 0.0)], "greedy": [(0.0, 0, 1.0, 0.0)],
         "mixed": [(0.8, 50, 0.95, 0.02), (1.0, 0, 0.9, 0.0), (0.0, 0, 1.0, 0.0), (0.6, 1000, 1.0, 0.0),
                   (1.3, 0, 1.0, 0.05), (1.0, 0, 1.0, 0.0), (0.7, 20, 0.8, 0.0)]}


def prepare_sample(case, seed):
    s, i = State(case), Inputs(seed)
    rows, count = case["rows"], case["count"]
    # A model's logits: a broad bulk and a few tokens well above it.
    s.logits = 2.5 * i.normal(rows, count)
    likely = (i.uniform(rows, 24) * count).long().clamp_(max=count - 1)
    s.logits.scatter_add_(1, likely, 6.0 + 8.0 * i.uniform(rows, 24))
    s.uniform = i.uniform(rows)
    rule = [RULES[case["rule"]][r % len(RULES[case["rule"]])] for r in range(rows)]
    s.temperature, s.top_p, s.min_p = (torch.tensor([r[k] for r in rule], device=DEVICE, dtype=torch.float32) for k in (0, 2, 3))
    s.top_k = torch.tensor([r[1] for r in rule], device=DEVICE, dtype=torch.int32)
    # The same as the records that a server uploads.
    s.params = torch.stack([s.temperature.view(torch.int32), s.top_k, s.top_p.view(torch.int32), s.min_p.view(torch.int32)], 1).contiguous()
    s.ids = torch.zeros(rows, device=DEVICE, dtype=torch.int32)
    return s


def sample_plain(s):
    """Sorted rows and running sums, in 64 bits: a draw next to a border of
    two tokens goes by the last bits of the sums."""
    count = s.logits.shape[1]
    value, index = torch.sort(s.logits, dim=1, descending=True, stable=True)
    greedy = ~(s.temperature > 0)
    heat = torch.where(greedy, 1.0, s.temperature).double()[:, None]
    value = value.double()
    weight = torch.exp((value - value[:, :1]) / heat)
    rank = torch.arange(count, device=DEVICE)
    top_k = s.top_k[:, None]
    weight = torch.where((top_k <= 0) | (rank < top_k), weight, 0.0)
    top_p = s.top_p.double()[:, None]
    run = torch.cumsum(weight, 1)
    keep = (top_p >= 1) | (run - weight < top_p * run[:, -1:]) | (rank == 0)
    keep &= (weight >= s.min_p.double()[:, None]) | (rank == 0)
    weight = torch.where(keep, weight, 0.0)
    run = torch.cumsum(weight, 1)
    over = run > s.uniform.double()[:, None] * run[:, -1:]
    pick = torch.where(greedy, 0, over.int().argmax(1))
    return index.gather(1, pick[:, None])[:, 0].int()


def sample_own(s):
    context().sample_rows(s.logits.data_ptr(), s.case["rows"], s.case["count"], s.params.data_ptr(), s.uniform.data_ptr(),
                          s.ids.data_ptr())
    return s.ids


def exact_sample(case, seed):
    s = prepare_sample(case, seed)
    logits, u = s.logits.cpu().numpy().astype(np.float64), s.uniform.cpu().numpy().astype(np.float64)
    heat, top_k = s.temperature.cpu().numpy().astype(np.float64), s.top_k.cpu().numpy()
    top_p, min_p = s.top_p.cpu().numpy().astype(np.float64), s.min_p.cpu().numpy().astype(np.float64)
    ids = np.zeros(case["rows"], np.int32)
    for r in range(case["rows"]):
        order = np.lexsort((np.arange(case["count"]), -logits[r]))
        if not heat[r] > 0:
            ids[r] = order[0]
            continue
        order = order[:top_k[r] or None]
        w = np.exp((logits[r][order] - logits[r][order[0]]) / heat[r])
        before = np.cumsum(w) - w
        if top_p[r] < 1:
            w = w[:max(1, int(np.sum(before < top_p[r] * w.sum())))]
        w = w[w >= min_p[r]]
        run = np.cumsum(w)
        ids[r] = order[min(int(np.searchsorted(run, u[r] * run[-1], side="right")), len(w) - 1)]
    return torch.from_numpy(ids)


def work_sample(case):
    return {"bytes": case["rows"] * (4 * case["count"] + 24), "flops": 0}


# ---------------------------------------------------------------------------
KINDS = {"attend": (prepare_attend, attend_plain, attend_own, exact_attend, work_attend),
         "append": (prepare_append, append_plain, append_own, exact_append, work_append),
         "copy": (prepare_copy, copy_plain, copy_own, exact_copy, work_copy),
         "sample": (prepare_sample, sample_plain, sample_own, exact_sample, work_sample)}


def prepare(case, seed):
    s = KINDS[case["kind"]][0](case, seed)
    if own:
        # The package's context has a stream of its own, which does not wait
        # for what torch's still has queued for the inputs.
        torch.cuda.synchronize()
    return s


def run(state):
    """One pass. With `own` set its outputs are written on the context's
    stream: whoever reads them on another waits for the context
    (`context().sync()`) or the device first."""
    return KINDS[state.case["kind"]][2 if own else 1](state)


def exact(case, seed):
    return KINDS[case["kind"]][3](case, seed)


def work(case):
    return KINDS[case["kind"]][4](case)
