"""How many bits of a query and of a softmax weight reach the products of
zg_paged_attn_device over a ZG_BF16 cache: three bfloat16 parts of 32-bit
queries and of the weights of 32-bit outputs, 24 bits in all, two parts of the
weights of 16-bit outputs.  The inputs are built so that the last part decides
and every other rounding is small beside it; the CPU tests show that one part
less would not pass the limits that the GPU tests set."""
import numpy as np
import pytest
import torch

import paged_reference as ref
from paged_reference import U
from zerogravity_amd import _lib as L

F32, BF16 = torch.float32, torch.bfloat16
LOG2E = np.float32(1.4426950408889634)
# the scale that times log2(e) is 1 in 32 bits: queries enter the products as they are
ONE = next(s for s in (np.float32(np.log(2)), np.nextafter(np.float32(np.log(2)), np.float32(1)),
                       np.nextafter(np.float32(np.log(2)), np.float32(0))) if np.float32(s * LOG2E) == 1)


def parts(x, n):
    """The sum of a float32 tensor's first n bfloat16 parts, each the first 8 bits of what is left."""
    left, total = x.clone(), torch.zeros_like(x, dtype=torch.float64)
    for _ in range(n):
        high = (left.view(torch.int32) & -65536).view(F32)
        total += high.double()
        left = left - high
    return total


def in_parts(q, keys, values, scale, of_query, of_weight):
    """softmax_rows with that many parts of a query and of a weight (the
    weights' sum is taken in full), 64 bits otherwise."""
    log2 = float(np.float32(scale) * LOG2E)
    query = parts(q * np.float32(log2), of_query) if q.dtype == F32 else q.double() * log2
    out = torch.zeros(q.shape, dtype=torch.float64)
    group = q.shape[0] // keys.shape[1]
    for h in range(q.shape[0]):
        k, v = keys[:, h // group].double(), values[:, h // group].double()
        s = k @ query[h]
        w = torch.exp2(s - s.max()).float()
        out[h] = parts(w, of_weight) @ v / w.double().sum()
    return out


def place(b, rows, keys, values):
    """Writes the prefix's and row r's own keys and values (rows[r] of them)
    into a Batch's pages and its reference."""
    def put(pages, k, v):
        i = torch.arange(k.shape[0])
        b.keys[pages.long()[i // b.page], i % b.page] = k.to(b.keys.dtype)
        b.values[pages.long()[i // b.page], i % b.page] = v.to(b.values.dtype)
        return k.double(), v.double()
    n = b.prefix_tokens
    b.shared = put(b.prefix, keys[:n], values[:n])
    b.own = [put(b.table[r], keys[n:n + max(m, 0)], values[n:n + max(m, 0)]) for r, m in enumerate(rows)]


def last_bits_of_queries(seed, rows, kv_heads, group, dim, prefix, lengths):
    """Pairs of elements s (1 + 2^-8 + d) and -s (1 + 2^-8), d of 8 bits below
    2^-15: the third part of the first.  A key is 2^16 at one pair, so the
    first parts' products are +-2^16 and the second's +-2^8, which cancel
    within one product, and a score is s d 2^16 = +-m / 128, m < 256, exact in
    32 bits in any order."""
    b = ref.Batch(seed, rows, kv_heads, group, dim, 16, prefix, lengths, F32, BF16)
    g = torch.Generator().manual_seed(seed)
    d = torch.randint(1, 256, (rows, group * kv_heads, dim // 2), generator=g) * 2.0 ** -23
    sign = torch.randint(0, 2, d.shape, generator=g) * 2.0 - 1
    b.q = torch.stack([sign * (1 + 2.0 ** -8 + d), -sign * torch.full_like(d, 1 + 2.0 ** -8)], -1).view(rows, -1, dim)
    total = prefix + max(max(lengths), 0)
    pair = torch.randint(0, dim // 2, (total, kv_heads), generator=g)
    keys = torch.zeros(total, kv_heads, dim // 2, 2)
    keys[torch.arange(total)[:, None], torch.arange(kv_heads), pair] = 2.0 ** 16
    values = torch.randn(total, kv_heads, dim, generator=g).to(BF16).float()
    place(b, lengths, keys.view(total, kv_heads, dim), values)
    b.scale = float(ONE)
    return b


def limit_of_scores(out, mass, tokens):
    """Exact scores of at most 2 in log2: a weight is off by the scale's
    rounding (2 U times a score of 2 ln 2) and the exponential's (2 U), and by
    what a reference other than the maximum adds (2 U for each of three
    rescalings); sums and joins add a rounding for each token and piece."""
    return (2 * tokens + 64) * U * mass + 2 * U * out.abs()


def few_that_weigh(seed, rows, kv_heads, group, dim, prefix, lengths, live, io, signs):
    """Of the tokens that a row sees only `live` successive ones, in one tile,
    weigh anything; their values are 1 (or +-1), so an output is 1 (or a sum
    of +-weights).  The others' last element makes their score -2^14."""
    b = ref.Batch(seed, rows, kv_heads, group, dim, 16, prefix, lengths, io, BF16)
    g = torch.Generator().manual_seed(seed)
    total = prefix + max(max(lengths), 0)
    keys = torch.randn(total, kv_heads, dim, generator=g).to(BF16).float()
    values = torch.randn(total, kv_heads, dim, generator=g).to(BF16).float()
    keys[..., -1] = -2.0 ** 14
    at = (prefix // 2 if prefix else min(n for n in lengths if n > 0) // 2) // 32 * 32 + 5
    keys[at:at + live, :, -1] = 0.0
    values[at:at + live] = 1.0
    if signs:
        values[at:at + live] = torch.randint(0, 2, (live, kv_heads, dim), generator=g) * 2.0 - 1
        b.q = b.q * 0.125  # weights near each other, so that sums of both signs are small
    b.q[..., -1] = 16.0  # times 2^14 and a scale of at least 1 / 16
    place(b, lengths, keys, values)
    b.live = (at, live)
    return b


# rows, kv heads, group, dim, prefix, own lengths: rows' own tiles; the prefix by 16 queries; by 128 (more than 6144
# tiles of 16 queries: 40 blocks of 16 over 165 tiles, 80 over 79); both at once
CASES = [(9, 2, 4, 256, 0, [700, 64, 33, 257, 40, 2000, 129, 90, 65]), (3, 1, 16, 64, 0, [5000, 96, 41]),
         (5, 4, 5, 128, 700, [0] * 5), (16, 2, 4, 256, 600, [0] * 16), (40, 1, 16, 64, 5280, [0] * 40),
         (80, 2, 8, 128, 2528, [0] * 80), (40, 1, 16, 256, 5280, [0] * 40), (33, 1, 16, 128, 6400, [(r * 7) % 50 for r in range(33)])]


@pytest.fixture(scope="module")
def ctx():
    c = L.Context(0)
    yield c
    c.close()


def attend(ctx, b):
    from test_paged_attn_gpu import Device
    return Device(b).attend(ctx).double().cpu()


def some(rows):
    return sorted({0, 1, 2, rows // 2, rows - 1} & set(range(rows)))


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES)
def test_queries_enter_in_24_bits(ctx, case):
    b = last_bits_of_queries(7, *case)
    got = attend(ctx, b)
    for r in some(case[0]):
        want, mass, _, tokens = b.reference(r)
        assert ((got[r] - want).abs() <= limit_of_scores(want, mass, tokens)).all(), r


@pytest.mark.parametrize("case", CASES)
def test_two_parts_of_a_query_would_not_do(case):
    """Nor would 32-bit scores of queries rounded to 16 bits: the limit holds
    three parts only."""
    b = last_bits_of_queries(7, *case)
    for r in some(case[0]):
        want, mass, _, tokens = b.reference(r)
        limit = limit_of_scores(want, mass, tokens)
        keys, values = (torch.cat([s, o]) for s, o in zip(b.shared, b.own[r]))
        assert ((in_parts(b.q[r], keys, values, b.scale, 3, 3) - want).abs() <= limit).all()
        if tokens > 1:
            assert ((in_parts(b.q[r], keys, values, b.scale, 2, 3) - want).abs() > limit).double().mean() > 0.5, r


LIVE = 4


def limit_of_weights():
    """Outputs that are a sum of LIVE weights over the same sum: each weight's
    three parts and the sum of weights add 4 roundings a token, the division
    and the joins 8 more."""
    return (4 * LIVE + 8) * U


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES)
def test_weights_enter_in_24_bits(ctx, case):
    b = few_that_weigh(8, *case, LIVE, F32, False)
    got = attend(ctx, b)
    assert ((got - 1).abs() <= limit_of_weights()).all(), float((got - 1).abs().max() / U)


@pytest.mark.parametrize("case", CASES)
def test_two_parts_of_a_weight_would_not_do(case):
    b = few_that_weigh(8, *case, LIVE, F32, False)
    off = []
    for r in some(case[0]):
        keys, values = (torch.cat([s, o]) for s, o in zip(b.shared, b.own[r]))
        assert ((in_parts(b.q[r], keys, values, b.scale, 3, 3) - 1).abs() <= limit_of_weights()).all()
        off.append((in_parts(b.q[r], keys, values, b.scale, 3, 2) - 1).abs())
    assert (torch.cat(off) > limit_of_weights()).double().mean() > 0.5


def limit_of_16_bits(want, mass):
    """Two parts leave out 2^-16 of each weight at most, so 2^-16 of sum w |v|,
    whatever is left of it after the signs; scores of 16-bit queries are sums
    in 32 bits, sum |q||k| scale < 4, 256 U of it at most; one rounding to
    bfloat16 of a value that is off by that."""
    return (2.0 ** -16 + 2 * 4 * 256 * U) * mass + 1.01 * ref.half_step(BF16) * want.abs()


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES)
def test_weights_of_16_bit_outputs_enter_in_two_parts(ctx, case):
    b = few_that_weigh(9, *case, 2, BF16, True)
    got = attend(ctx, b)
    for r in some(case[0]):
        want, mass, _, _ = b.reference(r)
        assert ((got[r] - want).abs() <= limit_of_16_bits(want, mass)).all(), r


def test_one_part_of_a_weight_would_not_do():
    beside = []
    for case in CASES:
        b = few_that_weigh(9, *case, 2, BF16, True)
        for r in some(case[0]):
            want, mass, _, _ = b.reference(r)
            limit = limit_of_16_bits(want, mass)
            keys, values = (torch.cat([s, o]) for s, o in zip(b.shared, b.own[r]))
            at, live = b.live
            near = keys[at:at + live].abs().repeat_interleave(case[2], 1) * b.q[r].double().abs()
            assert (near.sum(-1) * b.scale < 4).all()  # what the limit takes for granted
            two, one = (in_parts(b.q[r], keys, values, b.scale, 1, n).to(BF16).double() for n in (2, 1))
            assert ((two - want).abs() <= limit).all()
            beside.append(((one - want).abs() > limit).double().flatten())
    assert torch.cat(beside).mean() > 0.1
