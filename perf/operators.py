"""The paged cache's and the readout's operators, as cases that can be timed and checked.

Three operators of a batch that decodes over a KV cache in pages:

* append: a token's query and key normalised per head and rotated to its
  position, its key and value stored in the page that holds the position
  (zg_paged_append_device);
* attend: each row's query over a prefix that all rows share, in pages of its
  own, and then over the row's own pages (zg_paged_attn_device);
* adjust: penalties for repeated tokens, biases and a grammar's mask on the
  logits, and the highest one left (zg_logits_adjust_device).

`own` says which side `run` computes: the operators in plain torch, or the
library's kernels.  Head layouts are those of the 2B- and 0.8B-shaped models
(8 query and 2 KV heads of 256, 64 dimensions rotated) and others of the kind.
"""
import functools
import math

import numpy as np
import torch

own = False

DEV = "cuda"
EPS = 1e-6
VOCAB = 151936
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
CODES = {"f32": 0, "bf16": 30}  # the library's type codes


def theta_scale(rotate):
    """The frequencies' ratio, in the 32 bits that the entry point takes."""
    return float(np.float32(1e7 ** (-2.0 / rotate)))


def listed():
    layout = dict(q_heads=8, kv_heads=2, head_dim=256)
    return [
        # one request decoding, a layer's append: nothing but latency
        dict(name="append_1row", op="append", **layout, rotate=64, tokens=1, rows=1, first=2047, page=16, io="f32",
             kv="bf16", norm=True),
        # the same of a full batch
        dict(name="append_32rows", op="append", **layout, rotate=64, tokens=32, rows=32, first=2048, page=16,
             io="f32", kv="bf16", norm=True),
        # a long prompt's keys and values of one layer
        dict(name="append_prompt_8192", op="append", **layout, rotate=64, tokens=8192, rows=1, first=0, page=64,
             io="f32", kv="bf16", norm=True),
        # three requests' prompt chunks in one call, far into a long context, 16-bit activations, odd pages
        dict(name="append_chunks_777", op="append", q_heads=20, kv_heads=4, head_dim=128, rotate=128, tokens=777,
             rows=3, first=200000, page=7, io="bf16", kv="f32", norm=False),
        # one request decoding after a prompt of 2048 tokens
        dict(name="attend_1row_2048", op="attend", **layout, rows=1, prefix=0, shortest=2048, longest=2048, page=16,
             io="f32", kv="bf16"),
        # a batch that shares a system prompt, each row some way into its answer
        dict(name="attend_32rows_prefix_2048", op="attend", **layout, rows=32, prefix=2048, shortest=1, longest=512,
             page=16, io="f32", kv="bf16"),
        # unrelated requests of very different lengths, some just admitted without a token
        dict(name="attend_24rows_ragged", op="attend", **layout, rows=24, prefix=0, shortest=0, longest=16384,
             page=64, io="bf16", kv="bf16"),
        # many answers to one long document
        dict(name="attend_64rows_prefix_32768", op="attend", **layout, rows=64, prefix=32768, shortest=1,
             longest=1024, page=64, io="f32", kv="bf16"),
        # a cache held in 32 bits, five query heads to a KV head, odd lengths and pages
        dict(name="attend_9rows_f32_cache", op="attend", q_heads=20, kv_heads=4, head_dim=128, rows=9, prefix=1501,
             shortest=3, longest=701, page=13, io="f32", kv="f32"),
        # the readout of one request, of a batch and of the largest batch
        dict(name="adjust_1row", op="adjust", rows=1, vocab=VOCAB, history=600, biases=5, masked=True, io="f32"),
        dict(name="adjust_32rows", op="adjust", rows=32, vocab=VOCAB, history=2500, biases=40, masked=True, io="f32"),
        dict(name="adjust_64rows_bf16", op="adjust", rows=64, vocab=VOCAB, history=9000, biases=300, masked=False,
             io="bf16"),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["append", "attend", "attend", "adjust"])
    if op == "adjust":
        return dict(op=op, rows=log(1, 64), vocab=rng.choice([VOCAB, log(1000, VOCAB)]), history=log(1, 16384),
                    biases=rng.choice([0, log(1, 300)]), masked=rng.random() < 0.6, io=rng.choice(["f32", "f32", "bf16"]))
    group, kv_heads, head_dim = rng.choice([(4, 2, 256), (4, 2, 256), (4, 1, 256), (1, 8, 128), (5, 4, 128),
                                            (8, 2, 64), (16, 1, 128), (7, 3, 64)])
    case = dict(op=op, q_heads=group * kv_heads, kv_heads=kv_heads, head_dim=head_dim)
    kinds = dict(page=log(1, 256), io=rng.choice(["f32", "f32", "bf16"]), kv=rng.choice(["bf16", "bf16", "f32"]))
    # how much more a token costs than in the listed layout of 8 and 2 heads of 256
    more = max(1.0, group * kv_heads * head_dim / 2048, kv_heads * head_dim / 512 * (2 if kinds["kv"] == "f32" else 1))
    if op == "append":
        tokens = log(1, rng.choice([64, int(8192 / more)]))
        return dict(case, rotate=rng.choice([head_dim // 4, head_dim, 64]), tokens=tokens,
                    rows=min(tokens, log(1, 64)), first=rng.choice([0, log(1, 500000)]), norm=rng.random() < 0.5,
                    **kinds)
    rows = log(1, 64)
    longest = log(1, int(min(16384, 65536 / rows) / more))
    return dict(case, rows=rows, prefix=rng.choice([0, log(1, int(32768 / more)), log(1, 4096)]),
                shortest=rng.choice([0, 1, longest]), longest=longest, **kinds)


# ------------------------------------------------------------------- inputs

class Source:
    """Random inputs on the GPU, made from one seed."""

    def __init__(self, seed):
        self.g = torch.Generator(device=DEV)
        self.g.manual_seed(seed)

    def normal(self, *shape, scale=1.0, mean=0.0, dtype=torch.float32):
        return (mean + scale * torch.randn(*shape, device=DEV, generator=self.g)).to(dtype)

    def uniform(self, *shape, lo=0.0, hi=1.0):
        return lo + (hi - lo) * torch.rand(*shape, device=DEV, generator=self.g)

    def below(self, hi, *shape):
        return torch.randint(0, hi, shape, device=DEV, generator=self.g)

    def order(self, n):
        return torch.randperm(n, device=DEV, generator=self.g)


def lengths_of(case):
    """The rows' own lengths, from the shortest to the longest in equal ratios."""
    lo, hi, n = case["shortest"], case["longest"], case["rows"]
    if n == 1:
        return [hi]
    return [lo if i == 0 else int(round(max(lo, 1) * (hi / max(lo, 1)) ** (i / (n - 1)))) for i in range(n)]


def pages_of(tokens, page):
    return -(-tokens // page)


def cache(case, src, pages):
    shape = (pages, case["page"], case["kv_heads"], case["head_dim"])
    return src.normal(*shape, dtype=DTYPES[case["kv"]]), src.normal(*shape, dtype=DTYPES[case["kv"]])


def prepare(case, seed):
    src = Source(seed)
    s = dict(case=case)
    if case["op"] == "adjust":
        rows, vocab, history = case["rows"], case["vocab"], case["history"]
        # a token is likelier the lower its rank, and ranks are dealt over the vocabulary
        ranks = (vocab ** src.uniform(rows, history) - 1).long().clamp_(0, vocab - 1)
        lengths = (history * (0.5 + 0.5 * src.uniform(rows))).ceil().int().clamp_(1, history)
        ids = src.order(vocab)[:max(1, case["biases"])].int().repeat(rows, 1)
        words = -(-vocab // 32)
        grammars = max(1, rows // 2)
        bits = src.below(1 << 32, grammars, words)
        bits |= src.below(1 << 32, grammars, words)
        bits[0] &= src.below(1 << 32, words) & src.below(1 << 32, words) & src.below(1 << 32, words)
        s.update(logits=src.normal(rows, vocab, scale=3.0, dtype=DTYPES[case["io"]]),
                 history=src.order(vocab)[ranks].int(), history_lengths=lengths,
                 prompts=(lengths * src.uniform(rows)).int(),
                 repetition=src.uniform(rows, lo=1.0, hi=1.5), frequency=src.uniform(rows, hi=0.7),
                 presence=src.uniform(rows, hi=0.7), bias_ids=ids,
                 bias_values=src.normal(rows, ids.shape[1], scale=4.0),
                 bias_lengths=torch.full((rows,), case["biases"], dtype=torch.int32, device=DEV),
                 masks=(bits - ((bits >> 31) << 32)).int(),
                 # every third row decodes without a grammar
                 mask_of=torch.tensor([-1 if r % 3 == 2 else r // 2 % grammars for r in range(rows)],
                                      dtype=torch.int32, device=DEV),
                 out=torch.empty(rows, vocab, dtype=DTYPES[case["io"]], device=DEV),
                 greedy=torch.empty(rows, dtype=torch.int32, device=DEV))
    elif case["op"] == "append":
        tokens, rows, page = case["tokens"], case["rows"], case["page"]
        counts = torch.bincount(torch.arange(tokens) % rows, minlength=rows)
        of = torch.repeat_interleave(torch.arange(rows), counts)
        at = torch.arange(tokens) - (torch.cumsum(counts, 0) - counts)[of]
        # only the pages that the call's tokens fall into are there: those of earlier tokens are another's
        held = pages_of(case["first"] + int(counts.max()), page)
        skip = case["first"] // page
        table = torch.full((rows, held), -1, dtype=torch.int32, device=DEV)
        table[:, skip:] = src.order(rows * (held - skip)).int().view(rows, -1)
        q, kv, d = case["q_heads"], case["kv_heads"], case["head_dim"]
        keys, values = cache(case, src, rows * (held - skip))
        s.update(proj=src.normal(tokens, (q + 2 * kv) * d, dtype=DTYPES[case["io"]]),
                 q_norm=src.normal(d, scale=0.1, mean=1.0), k_norm=src.normal(d, scale=0.1, mean=1.0),
                 positions=(case["first"] + at).int().to(DEV), of=of.int().to(DEV), table=table, keys=keys,
                 values=values, query=torch.empty(tokens, q * d, dtype=DTYPES[case["io"]], device=DEV))
    else:
        rows, page, prefix = case["rows"], case["page"], case["prefix"]
        lengths = lengths_of(case)
        shared, wide = pages_of(prefix, page), max(1, pages_of(max(lengths), page))
        needed = [pages_of(n, page) for n in lengths]
        ids = src.order(max(1, shared + sum(needed))).int()
        table = torch.full((rows, wide), -1, dtype=torch.int32)
        table[torch.arange(wide).view(1, -1) < torch.tensor(needed).view(-1, 1)] = ids[shared:shared + sum(needed)].cpu()
        keys, values = cache(case, src, ids.numel())
        mixed = src.order(rows)
        s.update(q=src.normal(rows, case["q_heads"] * case["head_dim"], scale=1.5, dtype=DTYPES[case["io"]]),
                 keys=keys, values=values, prefix_table=ids[:shared].contiguous(),
                 table=table.to(DEV)[mixed].contiguous(),
                 lengths=torch.tensor(lengths, dtype=torch.int32, device=DEV)[mixed].contiguous(),
                 out=torch.empty(rows, case["q_heads"] * case["head_dim"], dtype=DTYPES[case["io"]], device=DEV))
    torch.cuda.synchronize()
    return s


# -------------------------------------------------------------- plain forms

def normed(x, gamma):
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * gamma


def rotated(x, positions, rotate):
    """x [tokens, heads, head_dim], the pairs (i, i + rotate / 2) turned."""
    h = rotate // 2
    angle = positions.double().view(-1, 1, 1) * theta_scale(rotate) ** torch.arange(h, dtype=torch.float64, device=DEV)
    c, sn = torch.cos(angle).to(x.dtype), torch.sin(angle).to(x.dtype)
    a, b = x[..., :h], x[..., h:rotate]
    return torch.cat([a * c - b * sn, a * sn + b * c, x[..., rotate:]], -1)


def plain_append(s):
    case = s["case"]
    n, q, kv, d = case["tokens"], case["q_heads"], case["kv_heads"], case["head_dim"]
    heads = s["proj"].float().view(n, q + 2 * kv, d)
    query, key = heads[:, :q], heads[:, q:q + kv]
    if case["norm"]:
        query, key = normed(query, s["q_norm"]), normed(key, s["k_norm"])
    at = s["positions"].long()
    pages = s["table"][s["of"].long(), at // case["page"]].long()
    s["keys"][pages, at % case["page"]] = rotated(key, at, case["rotate"]).to(s["keys"].dtype)
    s["values"][pages, at % case["page"]] = heads[:, q + kv:].to(s["values"].dtype)
    return {"query": rotated(query, at, case["rotate"]).reshape(n, -1).to(s["proj"].dtype), "keys": s["keys"],
            "values": s["values"]}


def plain_attend(s):
    case = s["case"]
    rows, kv, d, prefix, page = case["rows"], case["kv_heads"], case["head_dim"], case["prefix"], case["page"]
    group = case["q_heads"] // kv
    q = s["q"].float().view(rows, kv, group, d) / math.sqrt(d)
    wide = s["table"].shape[1] * page

    def tokens(pool, table, n):  # [..., kv, n, d] of a table's first n tokens
        got = pool[table.long().clamp(min=0)].float().view(*table.shape[:-1], -1, kv, d)[..., :n, :, :]
        return got.transpose(-2, -3).contiguous()

    keys, values = (tokens(s[n], s["table"], wide) for n in ("keys", "values"))
    late = torch.arange(wide, device=DEV) >= s["lengths"].view(-1, 1, 1, 1)
    score = (q @ keys.transpose(-1, -2).contiguous()).masked_fill(late, -math.inf)
    if prefix:
        shared, shared_values = (tokens(s[n], s["prefix_table"], prefix) for n in ("keys", "values"))
        flat = q.transpose(0, 1).reshape(kv, rows * group, d)
        before = (flat @ shared.transpose(-1, -2).contiguous()).view(kv, rows, group, prefix).transpose(0, 1)
        score = torch.cat([before, score], -1)
    top = score.amax(-1, keepdim=True)
    weight = torch.exp(score - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = weight.sum(-1, keepdim=True)
    weight = weight / torch.where(total > 0, total, torch.ones_like(total))
    out = weight[..., prefix:].contiguous() @ values.masked_fill(late.transpose(-1, -2), 0.0)
    if prefix:
        part = weight[..., :prefix].transpose(0, 1).reshape(kv, rows * group, prefix) @ shared_values
        out = out + part.view(kv, rows, group, d).transpose(0, 1)
    return out.reshape(rows, -1).to(s["q"].dtype)


def plain_adjust(s):
    case = s["case"]
    rows, vocab = case["rows"], case["vocab"]
    x = s["logits"].double()
    at = torch.arange(case["history"], device=DEV)
    held = at < s["history_lengths"].view(-1, 1)
    answer = held & (at >= s["prompts"].view(-1, 1))
    zero = torch.zeros(rows, vocab, dtype=torch.int32, device=DEV)
    seen = zero.scatter_add(1, s["history"].long(), held.int()) > 0
    count = zero.scatter_add(1, s["history"].long(), answer.int())
    rep = s["repetition"].double().view(-1, 1)
    x = torch.where(seen, torch.where(x > 0, x / rep, x * rep), x)
    x = x - s["frequency"].double().view(-1, 1) * count - s["presence"].double().view(-1, 1) * (count > 0)
    if case["biases"]:
        x = x.scatter_add(1, s["bias_ids"].long(), s["bias_values"].double())
    if case["masked"]:
        bits = (s["masks"].unsqueeze(-1) >> torch.arange(32, dtype=torch.int32, device=DEV)) & 1
        allowed = bits.view(bits.shape[0], -1)[:, :vocab].bool()[s["mask_of"].long().clamp(min=0)]
        x = x.masked_fill(~(allowed | (s["mask_of"] < 0).view(-1, 1)), -math.inf)
    out = x.float().to(s["logits"].dtype)
    best = out == out.amax(-1, keepdim=True)
    first = torch.where(best, torch.arange(vocab, device=DEV), vocab).amin(-1)
    return {"logits": out, "greedy": first.int()}


# ---------------------------------------------------------- the kernels' side

CONTEXT = []


def context():
    """The program's one context, and the stream that its steps run on: torch's
    current one.  The library has no handle for torch's default stream, so a
    program that is still on that one moves to a stream of its own."""
    from zerogravity_amd import _lib as L
    if not CONTEXT:
        CONTEXT.extend([L.Context(0), torch.cuda.Stream()])
    stream = torch.cuda.current_stream()
    if not stream.cuda_stream:
        CONTEXT[1].wait_stream(stream)
        torch.cuda.set_stream(CONTEXT[1])
        stream = CONTEXT[1]
    return CONTEXT[0], stream


def p(t):
    return t.data_ptr()


def bind(s):
    """A state's call with its arguments in place, as a decode loop keeps it,
    for the stream that is then current."""
    from zerogravity_amd import _lib as L
    from zerogravity_amd import paged, sampling
    case, lib = s["case"], L.lib()
    ctx, stream = context()
    st = stream.cuda_stream
    for t in s.values():  # made before the program moved, perhaps
        if isinstance(t, torch.Tensor):
            t.record_stream(stream)
    if case["op"] == "adjust":
        rules = sampling.rules(history=s["history"], history_lengths=s["history_lengths"], prompt_lengths=s["prompts"],
                               repetition=s["repetition"], frequency=s["frequency"], presence=s["presence"],
                               bias_ids=s["bias_ids"] if case["biases"] else None, bias_values=s["bias_values"],
                               bias_lengths=s["bias_lengths"], masks=s["masks"] if case["masked"] else None,
                               mask_of=s["mask_of"])
        room = torch.empty(lib.zg_logits_adjust_workspace_bytes(case["rows"], case["vocab"]), dtype=torch.uint8,
                           device=DEV)
        s["call"] = functools.partial(
            lib.zg_logits_adjust_device, ctx.h, case["rows"], case["vocab"], p(s["logits"]), case["vocab"],
            CODES[case["io"]], rules, p(s["out"]), case["vocab"], p(s["greedy"]), 0, p(room), None, st)
        s["result"] = {"logits": s["out"], "greedy": s["greedy"]}
        s["kept"] = (rules, room)
        return
    pool = paged.cache(s["keys"], s["values"])
    size = s["proj" if case["op"] == "append" else "q"].element_size()
    if case["op"] == "append":
        rows = paged.rows(s["table"])
        q, kv, d = case["q_heads"], case["kv_heads"], case["head_dim"]
        wide = (q + 2 * kv) * d
        s["call"] = functools.partial(
            lib.zg_paged_append_device, ctx.h, pool, rows, case["tokens"], q, p(s["proj"]), wide, d,
            p(s["proj"]) + q * d * size, wide, p(s["proj"]) + (q + kv) * d * size, wide, CODES[case["io"]],
            p(s["q_norm"]) if case["norm"] else None, p(s["k_norm"]) if case["norm"] else None, EPS, case["rotate"],
            theta_scale(case["rotate"]), p(s["positions"]), p(s["of"]), p(s["query"]), None, st)
        s["result"] = {"query": s["query"], "keys": s["keys"], "values": s["values"]}
        s["kept"] = (pool, rows)
        return
    rows = paged.rows(s["table"], s["prefix_table"], case["prefix"])
    room = torch.empty(lib.zg_paged_attn_workspace_bytes(pool, rows, case["q_heads"]), dtype=torch.uint8, device=DEV)
    s["call"] = functools.partial(
        lib.zg_paged_attn_device, ctx.h, pool, rows, p(s["lengths"]), case["q_heads"], p(s["q"]),
        case["q_heads"] * case["head_dim"], CODES[case["io"]], 1.0 / math.sqrt(case["head_dim"]), p(room), p(s["out"]),
        case["q_heads"] * case["head_dim"], None, st)
    s["result"] = s["out"]
    s["kept"] = (pool, rows, room)


def run(s):
    if not own:
        return {"append": plain_append, "attend": plain_attend, "adjust": plain_adjust}[s["case"]["op"]](s)
    if "call" not in s:
        bind(s)
    CONTEXT[0].check(s["call"]())
    return s["result"]


# ------------------------------------------------------------- work, 64 bits

def work(case):
    if case["op"] == "adjust":
        rows, n = case["rows"], case["rows"] * case["vocab"]
        extra = rows * (case["history"] * 3 + case["biases"] * 8) + (max(1, rows // 2) * case["vocab"] / 8
                                                                     if case["masked"] else 0)
        return {"bytes": 2 * n * (4 if case["io"] == "f32" else 2) + extra, "flops": n}
    io, kv = (4 if case[k] == "f32" else 2 for k in ("io", "kv"))
    q, h, d = case["q_heads"], case["kv_heads"], case["head_dim"]
    if case["op"] == "append":
        n = case["tokens"]
        return {"bytes": n * d * (2 * q * io + 2 * h * (io + kv)), "flops": n * d * 8 * (q + h)}
    held = sum(lengths_of(case))
    return {"bytes": (case["prefix"] + held) * 2 * h * d * kv + 2 * case["rows"] * q * d * io,
            "flops": 4 * q * d * (case["rows"] * case["prefix"] + held)}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "adjust":
        return exact_adjust(case, s)
    q, kv, d, page = case["q_heads"], case["kv_heads"], case["head_dim"], case["page"]
    if case["op"] == "append":
        n = case["tokens"]
        heads = s["proj"].double().view(n, q + 2 * kv, d)
        if case["norm"]:
            gamma = torch.cat([s["q_norm"].double().repeat(q, 1), s["k_norm"].double().repeat(kv, 1)])
            turned = heads[:, :q + kv]
            turned = turned / (turned.pow(2).sum(-1, keepdim=True) / d + EPS).sqrt() * gamma
        else:
            turned = heads[:, :q + kv].clone()
        # each pair as a complex number, times the unit number of its angle
        h = case["rotate"] // 2
        angle = s["positions"].double()[:, None] * torch.pow(
            torch.tensor(theta_scale(case["rotate"]), dtype=torch.float64, device=DEV),
            torch.arange(h, dtype=torch.float64, device=DEV))
        pair = torch.complex(turned[..., :h], turned[..., h:2 * h]) * torch.polar(torch.ones_like(angle), angle)[:, None]
        turned = torch.cat([pair.real, pair.imag, turned[..., 2 * h:]], -1)
        keys, values = s["keys"].double(), s["values"].double()
        position, row = s["positions"].long(), s["of"].long()
        slot = s["table"].long()[row, torch.div(position, page, rounding_mode="floor")] * page + position % page
        keys.view(-1, kv, d).index_copy_(0, slot, turned[:, q:].contiguous())
        values.view(-1, kv, d).index_copy_(0, slot, heads[:, q + kv:].contiguous())
        return {"query": turned[:, :q].reshape(n, q * d), "keys": keys, "values": values}
    group = q // kv
    out = torch.zeros(case["rows"], kv, group, d, dtype=torch.float64, device=DEV)
    lengths, shared = s["lengths"].tolist(), pages_of(case["prefix"], page)
    for k in range(kv):
        first = [s[n][:, :, k][s["prefix_table"].long()].double().view(-1, d)[:case["prefix"]] if shared else
                 torch.empty(0, d, dtype=torch.float64, device=DEV) for n in ("keys", "values")]
        for r, n in enumerate(lengths):
            if n + case["prefix"] == 0:
                continue
            mine = s["table"][r, :pages_of(n, page)].long()
            key, value = (torch.cat([f, s[name][mine, :, k].double().reshape(-1, d)[:n]])
                          for f, name in zip(first, ("keys", "values")))
            query = s["q"][r].double().view(kv, group, d)[k]
            score = key @ query.t().contiguous() / math.sqrt(d)
            out[r, k] = torch.softmax(score, 0).t().contiguous() @ value
    return out.view(case["rows"], q * d)


def exact_adjust(case, s):
    """Row by row: what each seen, biased or forbidden token becomes."""
    rows, vocab = case["rows"], case["vocab"]
    x = s["logits"].double().cpu().numpy()
    h = {k: s[k].cpu().numpy() for k in ("history", "history_lengths", "prompts", "repetition", "frequency", "presence",
                                         "bias_ids", "bias_values", "masks", "mask_of")}
    for r in range(rows):
        tokens = h["history"][r, :h["history_lengths"][r]]
        seen = np.unique(tokens)
        rep = np.float64(h["repetition"][r])
        x[r, seen] = np.where(x[r, seen] > 0, x[r, seen] / rep, x[r, seen] * rep)
        made, count = np.unique(tokens[h["prompts"][r]:], return_counts=True)
        x[r, made] -= np.float64(h["frequency"][r]) * count + np.float64(h["presence"][r])
        if case["biases"]:
            np.add.at(x[r], h["bias_ids"][r], h["bias_values"][r].astype(np.float64))
        if case["masked"] and h["mask_of"][r] >= 0:
            bits = np.unpackbits(h["masks"][h["mask_of"][r]].view(np.uint8), bitorder="little")[:vocab]
            x[r, bits == 0] = -np.inf
    held = torch.from_numpy(x.astype(np.float32)).to(DTYPES[case["io"]]).float().numpy()
    return {"logits": torch.from_numpy(x).to(DEV), "greedy": torch.from_numpy(held.argmax(-1).astype(np.int32)).to(DEV)}
