"""The kernels of a cache held in 4 bits against plain computations: what is stored equals the plain form's bytes, what is read back is
exact, and attention is compared with 64 bits."""
import math

import pytest
import torch

import plain_kv4

pytestmark = pytest.mark.gpu

HALF_STEP = 2.0 ** -8                          # a rounding to bfloat16, relative


def lib(head_dim):
    from stratakv_b200.ops import kernels_for
    return kernels_for(torch.bfloat16, head_dim, verbose=False)


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def make_cache(kv, dim, block, lengths, fill=0xFF, spread=1.0, spare=3):
    """Paged codes and scales whose live rows hold random numbers; everything else is ``fill`` (0xFF: scales of NaN)."""
    width = max(1, -(-max(lengths) // block))
    total = len(lengths) * width + spare
    table = torch.randperm(total, device="cuda")[:len(lengths) * width].int().view(len(lengths), width).contiguous()
    cache = [torch.full((total, kv, block, w), fill, dtype=torch.uint8, device="cuda") for w in (dim // 2, dim // 2, dim // 16, dim // 16)]
    for s, length in enumerate(lengths):
        for of in (0, 1):
            codes, scale = plain_kv4.store(torch.randn(kv, length, dim, device="cuda") * spread)
            for b in range(-(-length // block)):
                rows = min(block, length - b * block)
                cache[of][table[s, b], :, :rows] = codes[:, b * block:b * block + rows]
                cache[2 + of][table[s, b], :, :rows] = scale[:, b * block:b * block + rows]
    return cache, table


def cached(cache, table, s, length, block, of):
    """Float64 ``[kv_heads, length, dim]``: keys (of 0) or values (of 1) of sequence s."""
    blocks = table[s, :-(-length // block)].long()
    return plain_kv4.read(cache[of][blocks], cache[2 + of][blocks]).transpose(0, 1).flatten(1, 2)[:, :length]


# ---- appending ---------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("heads,kv,dim,block,new,rotated", [
    (4, 2, 16, 16, [1], True), (3, 3, 80, 64, [5, 1, 70], True), (8, 2, 128, 32, [1] * 9, True), (7, 1, 64, 16, [33, 16, 15], False),
    (32, 8, 128, 64, [130], True), (5, 1, 208, 16, [3, 17], True), (2, 2, 256, 32, [31], False)])
def test_append_stores_the_plain_forms_bytes(heads, kv, dim, block, new, rotated):
    from stratakv_b200.parts.position import rope_table
    k = lib(dim)
    before = [7 * i + 3 for i in range(len(new))]
    lengths = [b + n for b, n in zip(before, new)]
    cache, table = make_cache(kv, dim, block, lengths, fill=0xA5)
    kept = [c.clone() for c in cache]
    n = sum(new)
    # loud and quiet groups, and some of zeros
    qkv = torch.randn(n, (heads + 2 * kv) * dim, device="cuda") * torch.exp2(torch.randint(-12, 9, (n, (heads + 2 * kv) * dim // 16), device="cuda").float()).repeat_interleave(16, 1)
    qkv[:, -16:] = 0.0
    positions = torch.cat([torch.arange(b, b + c) for b, c in zip(before, new)]).int().cuda()
    seqs = torch.repeat_interleave(torch.arange(len(new)), torch.tensor(new)).int().cuda()
    cos_sin = torch.from_numpy(rope_table(dim, 10000.0, max(lengths))).cuda() if rotated else None
    q_out = torch.full((n, heads * dim), float("nan"), device="cuda").bfloat16()
    k.append_kv4(qkv, cos_sin, positions, seqs, table, q_out, *cache, heads, kv, dim, block)
    rows = qkv.view(n, heads + 2 * kv, dim)
    turned = plain_kv4.rotate(rows[:, :heads + kv], cos_sin, positions)
    assert torch.equal(q_out, turned[:, :heads].flatten(1).bfloat16())
    blocks, at = table[seqs.long(), positions.long() // block].long(), positions.long() % block
    for of, x in ((0, turned[:, heads:]), (1, rows[:, heads + kv:])):
        codes, scale = plain_kv4.store(x)
        kept[of][blocks, :, at], kept[2 + of][blocks, :, at] = codes, scale
        # and what they stand for is the nearest of the numbers that their group's smallest sufficient scale has
        near = plain_kv4.read(codes, scale)
        step = plain_kv4.scale_table("cuda")[scale.long()].repeat_interleave(16, dim=-1)
        assert bool(((near - x.double()).abs() <= step * (0.5 + 2.0 ** -20)).all())
        assert bool((step * 7 * (1 + 2.0 ** -22) >= x.double().abs()).all())
    for mine, plain in zip(cache, kept):
        assert torch.equal(mine, plain)            # (nothing else was touched)


def test_append_at_the_borders_of_its_scales():
    """Groups whose largest number is 7 times a scale, and its neighbours; the largest and smallest numbers; what is not finite."""
    dim, block = 64, 16
    k = lib(dim)
    table64 = plain_kv4.scale_table()[1:plain_kv4.LARGEST + 1]
    exact = (table64 * 7).float()
    most = torch.cat([exact, torch.nextafter(exact, exact * 2), torch.nextafter(exact, exact * 0), torch.tensor([0.0, 1e-30, 1e-40, 6272.0, 6273.0, 1e9, 3.4e38])])
    n = -(-most.numel() // 4)
    values = torch.zeros(n, 4, 16)
    values.view(-1, 16)[:most.numel(), 3] = -most
    values.view(-1, 16)[:most.numel(), 7] = most * 0.5           # (half a step off two codes: ties go to the even one)
    qkv = torch.cat([torch.zeros(n, dim), torch.zeros(n, dim), values.flatten(1)], dim=1).cuda()
    special = qkv[:6].clone()
    special[:, dim:] = torch.randn(6, 2 * dim, device="cuda")
    for i, bad in enumerate([math.inf, -math.inf, math.nan, math.inf, math.nan, 1.0]):
        special[i, dim + 16 * (i % 4) + i] = bad
        special[i, 2 * dim + 5] = bad
    qkv = torch.cat([qkv, special]).contiguous()
    n = qkv.shape[0]
    cache, table = make_cache(1, dim, block, [n])
    q_out = torch.empty(n, dim, dtype=torch.bfloat16, device="cuda")
    k.append_kv4(qkv, None, torch.arange(n, device="cuda", dtype=torch.int32), torch.zeros(n, device="cuda", dtype=torch.int32), table, q_out,
                 *cache, 1, 1, dim, block)
    for of in (0, 1):
        codes, scale = plain_kv4.store(qkv[:, dim * (1 + of):dim * (2 + of)])
        blocks, at = table[0, torch.arange(n) // block].long(), torch.arange(n) % block
        assert torch.equal(cache[2 + of][blocks, 0, at], scale) and torch.equal(cache[of][blocks, 0, at], codes)
    out = [torch.empty(table.shape[1], 1, block, dim, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    k.unpack_kv4(*cache, table, ints([n]), *out, torch.empty_like(table), 1, dim, block)
    read = out[1].view(-1, dim)[:n].float().cpu()
    assert read[:n - 6].abs().max() == 6272.0 and bool(torch.isfinite(read[:n - 6]).all())
    assert bool(torch.isnan(read[n - 6:n - 1, :16]).all()) and bool(torch.isfinite(read[n - 1]).all()) and bool(torch.isfinite(read[n - 6:, 16:]).all())


def test_append_of_queries_alone_leaves_the_cache():
    k = lib(64)
    cache, table = make_cache(1, 64, 16, [20])
    kept = [c.clone() for c in cache]
    qkv = torch.randn(4, 4 * 64, device="cuda")
    q_out = torch.zeros(4, 128, dtype=torch.bfloat16, device="cuda")
    k.append_kv4(qkv, None, torch.arange(4, device="cuda", dtype=torch.int32), ints([0] * 4), table, q_out, *cache, 2, 1, 64, 16, write_kv=False)
    assert torch.equal(q_out, qkv[:, :128].bfloat16()) and all(torch.equal(a, b) for a, b in zip(cache, kept))


# ---- reading back ------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("kv,dim,block,lengths,keep,width", [
    (2, 16, 16, [1], 0, 1), (3, 80, 64, [64, 65, 1, 200], 0, 4), (1, 128, 16, [100, 17, 16, 33], 17, 3), (2, 64, 32, [130, 31], 1, 1),
    (2, 64, 32, [130, 31], 64, 3), (1, 256, 16, [40], 0, 5)])
def test_unpack_gives_what_the_codes_stand_for(kv, dim, block, lengths, keep, width):
    k = lib(dim)
    cache, table = make_cache(kv, dim, block, lengths)
    n = len(lengths)
    out = [torch.full((n * width, kv, block, dim), float("nan"), dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    out_table = torch.full_like(table, -7)
    k.unpack_kv4(*cache, table, ints(lengths), *out, out_table, kv, dim, block, keep)
    for s, length in enumerate(lengths):
        first = max(0, length - keep) // block if keep else 0
        for of in (0, 1):
            plain = cached(cache, table, s, length, block, of)
            wanted = torch.zeros(kv, width * block, dim, dtype=torch.float64, device="cuda")
            some = plain[:, first * block:first * block + width * block]
            wanted[:, :some.shape[1]] = some
            got = out[of].view(n, width, kv, block, dim)[s].transpose(0, 1).flatten(1, 2)
            assert torch.equal(got.double(), wanted)
        for b in range(table.shape[1]):
            assert int(out_table[s, b]) == (s * width + b - first if first <= b < first + width else 0)


# ---- attention ----------------------------------------------------------------------------------------------------------

def take(monkeypatch, few):
    """Whether steps read the 4-bit cache themselves or what unpack_kv4 gives."""
    from stratakv_b200.ops import Kernels
    monkeypatch.setattr(Kernels, "_kv4_few", staticmethod(lambda *sizes: few))
    monkeypatch.setattr(Kernels, "_kv4_plan", lambda self, *sizes: (self._kv4_prototyped or self._kv4_prototypes()) and None or self._kv4_plan_of(*sizes))


def check_attention(heads, kv, dim, block, before, new, window=0, spread=1.0, extra_rows=0, table_room=0):
    k = lib(dim)
    lengths = [b + n for b, n in zip(before, new)]
    cache, table = make_cache(kv, dim, block, lengths, spread=spread)
    if table_room:
        table = torch.cat([table, torch.zeros(table.shape[0], table_room, dtype=torch.int32, device="cuda")], dim=1).contiguous()
    tokens = sum(new)
    q = torch.randn(tokens + extra_rows, heads * dim, device="cuda").bfloat16()
    out = torch.full((tokens + extra_rows, heads * dim), 7.0, dtype=torch.bfloat16, device="cuda")
    cu = [0]
    for c in new:
        cu.append(cu[-1] + c)
    scale = 1.0 / math.sqrt(dim)
    wanted = k.attention_kv4_scratch(len(new), q.shape[0], max(new), table.shape[1], heads, kv, dim, block, window)
    scratch = torch.full((wanted,), 0xFF, dtype=torch.uint8, device="cuda")
    k.attention_kv4(q, *cache, table, ints(cu), ints(lengths), out, max(new), heads, kv, dim, block, scale, window, scratch)
    unpacked = k._kv4_plan(len(new), max(new), table.shape[1], heads, kv, dim, block, window)[0] > 0
    for s in range(len(new)):
        ref, sums, whole = plain_kv4.attention(q[cu[s]:cu[s + 1]].double().view(new[s], heads, dim), cached(cache, table, s, lengths[s], block, 0),
                                        cached(cache, table, s, lengths[s], block, 1), before[s], scale, window)
        got = out[cu[s]:cu[s + 1]].double().view(new[s], heads, dim)
        # The result is rounded once; a probability keeps 11 bits (8 behind unpack_kv4), its exponential and the
        # sums of products together another 2^-11 of what is added up.  A half below 2^-14 is a multiple of 2^-24: a probability, which is
        # held 2^7 times as large as it is next to the row's largest (the maximum in use is never above the largest), is off by at
        # most half of that over 2^7 there, 2^-32, and so is its key's share of the result next to a denominator of at least 1.
        # (Weights of nearly nothing show where the keys that have the weight hold zeros.)
        allowed = HALF_STEP * ref.abs() + ((2.0 ** -8 if unpacked else 2.0 ** -11) + 2.0 ** -11) * sums + 2.0 ** -32 * whole
        assert bool(((got - ref).abs() <= allowed).all()), (s, float(((got - ref).abs() / allowed).max()))
    assert bool((out[tokens:] == 7.0).all())


@pytest.mark.parametrize("heads,kv,dim,block,lengths,window", [
    (4, 2, 16, 16, [1], 0), (3, 3, 80, 64, [5, 64, 65, 130], 0), (8, 2, 128, 32, [1, 15, 16, 17, 300], 0), (32, 4, 64, 64, [2048, 3, 511], 0),
    (7, 1, 64, 16, [100, 257], 40), (24, 1, 128, 16, [77, 1000], 0), (32, 32, 128, 16, [200, 1, 45], 0), (2, 1, 208, 16, [129, 64], 0),
    (4, 1, 256, 64, [300], 17), (6, 2, 48, 32, [33, 500], 1), (32, 8, 128, 64, [9000], 1024), (2, 1, 192, 16, [70], 0)])
def test_attention_of_one_token_a_sequence(heads, kv, dim, block, lengths, window):
    check_attention(heads, kv, dim, block, [n - 1 for n in lengths], [1] * len(lengths), window)


@pytest.mark.parametrize("heads,kv,dim,block,before,new,window", [
    (8, 2, 128, 32, [0, 40, 100], [1, 3, 5], 0), (4, 4, 64, 16, [0, 7, 300], [16, 2, 9], 0), (3, 1, 80, 64, [62, 0], [5, 20], 0),
    (8, 1, 64, 64, [1000], [8], 33), (32, 8, 128, 16, [4000, 511], [5, 1], 0), (2, 1, 16, 48, [10], [70], 20), (2, 2, 208, 16, [3, 0], [9, 40], 0),
    (4, 2, 128, 48, [90], [50], 0), (4, 4, 128, 64, [700, 0], [96, 3], 0), (8, 1, 64, 16, [600, 10], [40, 1], 300)])
def test_attention_of_a_few_tokens_a_sequence(heads, kv, dim, block, before, new, window):
    check_attention(heads, kv, dim, block, before, new, window)


@pytest.mark.parametrize("heads,kv,dim,block,before,new,window", [
    (4, 2, 64, 64, [0], [300], 0), (4, 1, 128, 16, [77, 0, 900], [130, 1, 40], 0), (8, 8, 64, 32, [1000, 5], [65, 200], 100),
    (2, 1, 128, 128, [3], [513], 64), (8, 2, 64, 64, [0] * 5, [100, 1, 64, 65, 33], 0), (4, 4, 128, 64, [700, 0], [97, 96], 0),
    (8, 1, 64, 16, [600], [41], 0)])
@pytest.mark.parametrize("few", [False, True])
def test_attention_of_prompts(monkeypatch, heads, kv, dim, block, before, new, window, few):
    """Both ways, whichever the rule would take."""
    take(monkeypatch, few)
    check_attention(heads, kv, dim, block, before, new, window)


# (sequences so long that runs of chunks are dealt out, whose partial results a second launch adds up)
@pytest.mark.parametrize("heads,kv,dim,block,before,new,window", [
    (4, 2, 16, 16, [9000, 70], [1, 1], 0), (8, 1, 48, 64, [17000, 3], [1, 1], 0), (32, 4, 64, 64, [17000, 511], [1, 1], 0), (3, 3, 80, 16, [9000, 0], [6, 2], 0),
    (16, 2, 128, 64, [17000, 40], [1, 3], 0), (8, 8, 128, 16, [40, 9000], [1, 1], 0), (2, 1, 208, 16, [9000, 1], [1, 1], 0), (4, 1, 256, 64, [18000, 50], [1, 1], 17000),
    (24, 1, 64, 16, [9000, 17], [1, 2], 8500), (6, 2, 192, 64, [1, 17000], [1, 4], 0), (32, 8, 128, 64, [40000], [1], 0), (4, 4, 64, 64, [100_000], [1], 0)])
def test_attention_by_runs(heads, kv, dim, block, before, new, window):
    width = -(-max(b + n for b, n in zip(before, new)) // block)
    assert lib(dim).attention_kv4_scratch(len(new), sum(new), max(new), width, heads, kv, dim, block, window) > 0
    check_attention(heads, kv, dim, block, before, new, window)


def test_a_cluster_for_every_item_needs_no_scratch():
    """One block, a few, several waves of single ones."""
    for sizes in ((1, 1, 1, 4, 2, 64, 16), (1, 1, 30, 4, 2, 64, 64), (8, 1, 60, 32, 8, 64, 64), (100, 1, 5, 32, 4, 64, 64), (3, 9, 20, 8, 2, 64, 32)):
        assert lib(64).attention_kv4_scratch(sizes[0], sizes[0] * sizes[1], *sizes[1:]) == 0
    check_attention(32, 4, 64, 64, [290 + i % 30 for i in range(100)], [1] * 100)
    check_attention(8, 8, 128, 16, [(37 * i) % 150 for i in range(64)], [1 + i % 2 for i in range(64)])


@pytest.mark.parametrize("new", [[1, 1], [4, 2], [100, 30]])
def test_attention_leaves_rows_behind_the_last_sequence(monkeypatch, new):
    take(monkeypatch, new[0] < 100)
    check_attention(4, 2, 64, 32, [3000, 600], new, extra_rows=5, table_room=3)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("spread", [1e-4, 40.0])
def test_attention_over_quiet_and_loud_caches(dim, spread):
    """Scores of nearly nothing, and scores that leave one key (whose neighbours' probabilities vanish)."""
    check_attention(4, 1, dim, 16, [700, 40], [1, 1], spread=spread)


def run_step(k, q, cache, table, cu, ctx, heads, kv, dim, block, most, window=0):
    out = torch.empty_like(q)
    scratch = torch.full((k.attention_kv4_scratch(len(ctx), q.shape[0], most, table.shape[1], heads, kv, dim, block, window),), 0xFF, dtype=torch.uint8, device="cuda")
    k.attention_kv4(q, *cache, table, ints(cu), ints(ctx), out, most, heads, kv, dim, block, 1.0 / math.sqrt(dim), window, scratch)
    return out


@pytest.mark.parametrize("dim", [64, 128, 80])
@pytest.mark.parametrize("at", [0, 500, 998])
def test_what_is_not_finite_reaches_the_rows_that_see_it_alone(dim, at):
    """A value's NaN in one group of one position: only that group's numbers, only of queries at or behind that position; a key's NaN
    reaches all of such a query's numbers.  With a window, queries that have left it behind stay clean."""
    k = lib(dim)
    heads, kv, block, before, new = 4, 2, 16, 995, 5
    cache, table = make_cache(kv, dim, block, [before + new])
    q = torch.randn(new, heads * dim, device="cuda").bfloat16()
    clean = run_step(k, q, cache, table, [0, new], [before + new], heads, kv, dim, block, new, window=997)
    entry = table[0, at // block].long()
    spoiled = [c.clone() for c in cache]
    spoiled[3][entry, 1, at % block, 2] = plain_kv4.NOT_FINITE
    got = run_step(k, q, spoiled, table, [0, new], [before + new], heads, kv, dim, block, new, window=997).view(new, heads, dim)
    sees = torch.tensor([at <= before + i and at > before + i - 997 for i in range(new)])
    wanted = torch.zeros(new, heads, dim, dtype=torch.bool)
    wanted[:, 2:, 32:48] = sees[:, None, None]
    assert torch.equal(torch.isnan(got).cpu(), wanted)
    assert torch.equal(got[~wanted.cuda()], clean.view(new, heads, dim)[~wanted.cuda()])
    spoiled = [c.clone() for c in cache]
    spoiled[2][entry, 0, at % block, 1] = plain_kv4.NOT_FINITE
    got = run_step(k, q, spoiled, table, [0, new], [before + new], heads, kv, dim, block, new, window=997).view(new, heads, dim)
    wanted = torch.zeros(new, heads, dim, dtype=torch.bool)
    wanted[:, :2] = sees[:, None, None]
    assert torch.equal(torch.isnan(got).cpu(), wanted)
    assert torch.equal(got[~wanted.cuda()], clean.view(new, heads, dim)[~wanted.cuda()])


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_a_query_that_is_not_finite_gives_nan_and_spoils_no_other(bad):
    k = lib(64)
    cache, table = make_cache(1, 64, 16, [600, 600])
    q = torch.randn(2, 4 * 64, device="cuda").bfloat16()
    clean = run_step(k, q, cache, table, [0, 1, 2], [600, 600], 4, 1, 64, 16, 1)
    q[0, 64 + 3] = bad
    got = run_step(k, q, cache, table, [0, 1, 2], [600, 600], 4, 1, 64, 16, 1)
    assert bool(torch.isnan(got[0, 64:128]).all())
    got[0, 64:128] = clean[0, 64:128]
    assert torch.equal(got, clean)


def twice_off(cache, unpacked):
    """How far two results over this cache may lie apart before they are rounded: each is off by the roundings of its probabilities and its
    sums (see check_attention) times the largest value."""
    values = plain_kv4.read(cache[1], cache[3])
    return 2 * ((2.0 ** -8 if unpacked else 2.0 ** -11) + 2.0 ** -11) * float(values[~torch.isnan(values)].abs().max())


@pytest.mark.parametrize("new", [1, 4, 200])
def test_windows_of_any_size(monkeypatch, new):
    """One as long as what is cached, or longer, changes nothing; a negative one is refused, whichever way the step takes."""
    from stratakv_b200.ops import KernelError
    k = lib(64)
    cache, table = make_cache(2, 64, 16, [300 + new])
    q = torch.randn(new, 4 * 64, device="cuda").bfloat16()
    take(monkeypatch, new < 200)
    plain = run_step(k, q, cache, table, [0, new], [300 + new], 4, 2, 64, 16, new)
    for window in (300 + new, 10 ** 6, 2 ** 31 - new, 2 ** 31 - 1, 2 ** 32 + 5):
        got = run_step(k, q, cache, table, [0, new], [300 + new], 4, 2, 64, 16, new, window=window)
        if window < table.numel() * 16:                    # (one that the table could leave is cut as windows are: sums in another order)
            torch.testing.assert_close(got.float(), plain.float(), rtol=2 * HALF_STEP, atol=twice_off(cache, new == 200))
        else:
            assert torch.equal(got, plain), window
    with pytest.raises(KernelError, match="must not be negative"):
        run_step(k, q, cache, table, [0, new], [300 + new], 4, 2, 64, 16, new, window=-1)


def test_queries_of_any_size():
    """Powers of two on a query and off the scale change nothing but the products' exponents."""
    k = lib(128)
    cache, table = make_cache(1, 128, 64, [333])
    q = torch.randn(1, 2 * 128, device="cuda").bfloat16()
    plain = run_step(k, q, cache, table, [0, 1], [333], 2, 1, 128, 64, 1)
    for power in (-90, -20, 30, 100):
        out = torch.empty_like(q)
        scratch = torch.empty(k.attention_kv4_scratch(1, 1, 1, table.shape[1], 2, 1, 128, 64), dtype=torch.uint8, device="cuda")
        k.attention_kv4((q.float() * 2.0 ** power).bfloat16(), *cache, table, ints([0, 1]), ints([333]), out, 1, 2, 1, 128, 64,
                        2.0 ** -power / math.sqrt(128), 0, scratch)
        assert torch.equal(out, plain), power


def test_a_long_context_beyond_32_bit_offsets():
    """Blocks whose bytes lie beyond 2^31 from the cache's start."""
    dim, kv, block = 128, 8, 64
    k = lib(dim)
    blocks = (2 ** 31 // (kv * block * dim // 2)) + 40
    cache = [torch.zeros(blocks, kv, block, w, dtype=torch.uint8, device="cuda") for w in (64, 64, 8, 8)]
    table = torch.arange(blocks - 8, blocks, device="cuda", dtype=torch.int32)[None].contiguous()
    length = 8 * block - 5
    for of in (0, 1):
        codes, scale = plain_kv4.store(torch.randn(8, kv, block, dim, device="cuda"))
        cache[of][blocks - 8:], cache[2 + of][blocks - 8:] = codes, scale
    q = torch.randn(1, 8 * dim, device="cuda").bfloat16()
    out = run_step(k, q, cache, table, [0, 1], [length], 8, kv, dim, block, 1)
    ref, sums, _ = plain_kv4.attention(q.double().view(1, 8, dim), cached(cache, table, 0, length, block, 0), cached(cache, table, 0, length, block, 1),
                                    length - 1, 1.0 / math.sqrt(dim))
    assert bool(((out.double().view(1, 8, dim) - ref).abs() <= HALF_STEP * ref.abs() + 2.0 ** -10 * sums).all())


def test_append_read_back_and_attend_together():
    """A prompt, then single tokens, as they would be used: each step's result equals attention over what the plain form stores."""
    from stratakv_b200.parts.position import rope_table
    heads, kv, dim, block = 8, 2, 64, 16
    k = lib(dim)
    cache, table = make_cache(kv, dim, block, [160, 160])
    cos_sin = torch.from_numpy(rope_table(dim, 10000.0, 160)).cuda()
    stored = [[], []]
    before = [0, 0]
    for new in ([100, 37], [1, 1], [3, 2], [1, 1], [40, 1]):
        n = sum(new)
        qkv = torch.randn(n, (heads + 2 * kv) * dim, device="cuda")
        positions = torch.cat([torch.arange(b, b + c) for b, c in zip(before, new)]).int().cuda()
        seqs = torch.repeat_interleave(torch.arange(2), torch.tensor(new)).int().cuda()
        q = torch.empty(n, heads * dim, dtype=torch.bfloat16, device="cuda")
        k.append_kv4(qkv, cos_sin, positions, seqs, table, q, *cache, heads, kv, dim, block)
        after = [b + c for b, c in zip(before, new)]
        cu = [0, new[0], n]
        out = run_step(k, q, cache, table, cu, after, heads, kv, dim, block, max(new))
        rows = qkv.view(n, heads + 2 * kv, dim)
        turned = plain_kv4.rotate(rows[:, :heads + kv], cos_sin, positions)
        for s in range(2):
            mine = slice(cu[s], cu[s + 1])
            stored[s].append([plain_kv4.read(*plain_kv4.store(x[mine])) for x in (turned[:, heads:], rows[:, heads + kv:])])
            keys, values = (torch.cat([piece[i] for piece in stored[s]]).transpose(0, 1) for i in (0, 1))
            ref, sums, _ = plain_kv4.attention(turned[mine, :heads].bfloat16().double(), keys, values, before[s], 1.0 / math.sqrt(dim))
            allowed = HALF_STEP * ref.abs() + (2.0 ** -8 + 2.0 ** -11) * sums
            assert bool(((out[mine].double().view(new[s], heads, dim) - ref).abs() <= allowed).all())
        before = after


def test_which_way_a_step_attends():
    """The rule: a few tokens read the cache itself, prompts the numbers it stands for."""
    k = lib(64)
    assert k._kv4_plan(1, 1, 100, 4, 2, 64, 64, 0)[0] == 0 and k._kv4_plan(1, 2000, 40, 4, 2, 64, 64, 0)[0] == 40
    assert k._kv4_plan(2, 900, 20, 8, 8, 64, 64, 100)[0] == min(20, (100 + 900 - 1 + 62) // 64 + 1)
    assert k._kv4_plan(1, 300, 5, 4, 2, 64, 64, 0)[0] == 0 and k._kv4_plan(8, 300, 5, 4, 2, 64, 64, 0)[0] == 5     # (tiles for the whole GPU)
    assert k._kv4_plan(1, 2000, 40, 4, 2, 64, 48, 0)[0] == 0               # (the prompt kernel wants blocks that are powers of two)
    assert lib(80)._kv4_plan(1, 2000, 40, 4, 2, 80, 64, 0)[0] == 0         # (and heads of 64 or 128)


@pytest.mark.parametrize("new", [[0, 1, 0, 1], [3, 0, 0, 2]])
def test_sequences_without_new_tokens(new):
    """They have no rows, and nothing of their cache is read."""
    k = lib(64)
    before = [100, 700, 40, 300]
    cache, table = make_cache(2, 64, 16, [b + n for b, n in zip(before, new)])
    q = torch.randn(sum(new), 4 * 64, device="cuda").bfloat16()
    cu = [0]
    for c in new:
        cu.append(cu[-1] + c)
    got = run_step(k, q, cache, table, cu, [b + n for b, n in zip(before, new)], 4, 2, 64, 16, max(new))
    for s in range(4):
        if new[s]:
            alone = run_step(k, q[cu[s]:cu[s + 1]].contiguous(), cache, table[s:s + 1].contiguous(), [0, new[s]], [before[s] + new[s]], 4, 2, 64, 16, new[s])
            torch.testing.assert_close(got[cu[s]:cu[s + 1]].float(), alone.float(), rtol=2 * HALF_STEP, atol=2.0 ** -10)


def test_lengths_that_contradict_the_call_spoil_no_other_sequence():
    """More new tokens than the call's maximum, a negative length, one beyond the table: that sequence's rows are anyone's guess."""
    k = lib(64)
    cache, table = make_cache(2, 64, 16, [90, 90, 90, 90, 90, 90])
    q = torch.randn(8, 4 * 64, device="cuda").bfloat16()
    cu, ctx = [0, 1, 4, 5, 6, 7, 8], [90, 90, -5, 33, 10 ** 6, 70]
    for window in (0, 1, 20):
        got = run_step(k, q, cache, table, cu, ctx, 4, 2, 64, 16, 1, window=window)
        for s in (0, 3, 5):
            alone = run_step(k, q[cu[s]:cu[s] + 1].contiguous(), cache, table[s:s + 1].contiguous(), [0, 1], [ctx[s]], 4, 2, 64, 16, 1, window=window)
            torch.testing.assert_close(got[cu[s]].float(), alone[0].float(), rtol=2 * HALF_STEP, atol=twice_off(cache, False))


@pytest.mark.parametrize("some", [1, 2])
@pytest.mark.parametrize("window", [0, 150])
def test_prompts_are_read_back_a_few_sequences_at_a_time(monkeypatch, some, window):
    """The same results from a scratch that holds one sequence, or two, as from one that holds all."""
    from stratakv_b200 import ops
    k = lib(64)
    heads, kv, block, before, new = 8, 2, 64, [900, 0, 40, 700, 3], [130, 200, 1, 65, 129]
    lengths = [b + n for b, n in zip(before, new)]
    cache, table = make_cache(kv, 64, block, lengths)
    cu = [0]
    for c in new:
        cu.append(cu[-1] + c)
    q = torch.randn(cu[-1], heads * 64, device="cuda").bfloat16()
    take(monkeypatch, False)
    whole = k.attention_kv4_scratch(5, cu[-1], 200, table.shape[1], heads, kv, 64, block, window)
    at_once = run_step(k, q, cache, table, cu, lengths, heads, kv, 64, block, 200, window)
    monkeypatch.setattr(ops, "KV4_UNPACKED", whole // 5 * some)
    assert k.attention_kv4_scratch(5, cu[-1], 200, table.shape[1], heads, kv, 64, block, window) == whole // 5 * some
    got = run_step(k, q, cache, table, cu, lengths, heads, kv, 64, block, 200, window)
    # (blocks of the prompt kernel may share a tile's keys where there are few: sums in another order)
    torch.testing.assert_close(got.float(), at_once.float(), rtol=2 * HALF_STEP, atol=twice_off(cache, True))


@pytest.mark.parametrize("n_seqs,most", [(1100, 1), (2051, 2)])
def test_more_sequences_than_a_launch_takes(n_seqs, most):
    k = lib(64)
    lengths = [1 + (7 * i) % 40 + most for i in range(n_seqs)]
    cache, table = make_cache(1, 64, 16, [max(lengths)] * 3)
    table = table[torch.arange(n_seqs, device="cuda") % 3].contiguous()    # (three caches, many readers)
    q = torch.randn(n_seqs * most, 2 * 64, device="cuda").bfloat16()
    got = run_step(k, q, cache, table, [most * i for i in range(n_seqs + 1)], lengths, 2, 1, 64, 16, most)
    for s in (0, 1, 1023, 1024, 1025, n_seqs - 1):
        mine = slice(most * s, most * (s + 1))
        ref, sums, _ = plain_kv4.attention(q[mine].double().view(most, 2, 64), cached(cache, table, s, lengths[s], 16, 0),
                                           cached(cache, table, s, lengths[s], 16, 1), lengths[s] - most, 0.125)
        assert bool(((got[mine].double().view(most, 2, 64) - ref).abs() <= HALF_STEP * ref.abs() + 2.0 ** -10 * sums).all())


def test_the_last_launch_may_be_cut_in_another_way():
    """1,024 sequences that need no scratch, and 19 that do."""
    k = lib(64)
    n_seqs, heads, kv, most = 1043, 64, 8, 2
    sizes = (most, 64, heads, kv, 16, 0)
    assert k.lib.skv_attention_kv4_scratch(1024, *sizes) == 0 and k.lib.skv_attention_kv4_scratch(19, *sizes) > 0
    cache, table = make_cache(kv, 64, 16, [1024, 1024])
    table = table[torch.arange(n_seqs, device="cuda") % 2].contiguous()
    lengths = [1024 - (13 * i) % 700 for i in range(n_seqs)]
    q = torch.randn(n_seqs * most, heads * 64, device="cuda").bfloat16()
    got = run_step(k, q, cache, table, [most * i for i in range(n_seqs + 1)], lengths, heads, kv, 64, 16, most)
    for s in (0, 1023, 1024, n_seqs - 1):
        mine = slice(most * s, most * (s + 1))
        ref, sums, _ = plain_kv4.attention(q[mine].double().view(most, heads, 64), cached(cache, table, s, lengths[s], 16, 0),
                                           cached(cache, table, s, lengths[s], 16, 1), lengths[s] - most, 0.125)
        assert bool(((got[mine].double().view(most, heads, 64) - ref).abs() <= HALF_STEP * ref.abs() + 2.0 ** -10 * sums).all())


def test_a_captured_step_follows_its_inputs():
    """A replayed graph reads lengths, tables and rows as they are then; two graphs with a scratch each, on another stream than the capture's."""
    k = lib(128)
    heads, kv, dim, block = 8, 2, 128, 32
    cache, table = make_cache(kv, dim, block, [2000, 900])
    q = torch.randn(2, heads * dim, device="cuda").bfloat16()
    ctx, cu = ints([1500, 300]), ints([0, 1, 2])
    wanted = k.attention_kv4_scratch(2, 2, 1, table.shape[1], heads, kv, dim, block)
    graphs = []
    for _ in range(2):
        out, scratch = torch.empty_like(q), torch.empty(wanted, dtype=torch.uint8, device="cuda")
        call = lambda: k.attention_kv4(q, *cache, table, cu, ctx, out, 1, heads, kv, dim, block, dim ** -0.5, 0, scratch)
        call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call()
        graphs.append((graph, out, scratch))
    side = torch.cuda.Stream()
    for lengths in ([1500, 300], [2000, 1], [33, 900]):
        ctx.copy_(ints(lengths))
        q.normal_()
        torch.cuda.synchronize()
        graphs[0][0].replay()
        with torch.cuda.stream(side):
            graphs[1][0].replay()
        torch.cuda.synchronize()
        eager = torch.empty_like(q)
        k.attention_kv4(q, *cache, table, cu, ctx, eager, 1, heads, kv, dim, block, dim ** -0.5, 0, torch.empty(wanted, dtype=torch.uint8, device="cuda"))
        assert torch.equal(graphs[0][1], eager) and torch.equal(graphs[1][1], eager)
        for s, length in enumerate(lengths):
            ref, sums, _ = plain_kv4.attention(q[s:s + 1].double().view(1, heads, dim), cached(cache, table, s, length, block, 0),
                                               cached(cache, table, s, length, block, 1), length - 1, dim ** -0.5)
            assert bool(((eager[s:s + 1].double().view(1, heads, dim) - ref).abs() <= HALF_STEP * ref.abs() + 2.0 ** -10 * sums).all())


def test_another_device_than_the_current_one_is_refused(monkeypatch):
    from stratakv_b200.ops import KernelError
    k = lib(64)
    cache, table = make_cache(1, 64, 16, [20])
    q = torch.zeros(1, 64, dtype=torch.bfloat16, device="cuda")
    run_step(k, q, cache, table, [0, 1], [20], 1, 1, 64, 16, 1)
    current = torch.cuda.current_device()
    scratch = torch.empty(1 << 16, dtype=torch.uint8, device="cuda")
    cu, ctx = ints([0, 1]), ints([20])
    monkeypatch.setattr(torch.cuda, "current_device", lambda: current + 1)
    with pytest.raises(KernelError, match="another device"):
        k.attention_kv4(q, *cache, table, cu, ctx, q.clone(), 1, 1, 1, 64, 16, 0.125, 0, scratch)


# ---- refusals -----------------------------------------------------------------------------------------------------------

def test_refusals():
    from stratakv_b200.ops import KernelError
    k = lib(64)
    cache, table = make_cache(2, 64, 16, [40])
    q = torch.zeros(1, 4 * 64, dtype=torch.bfloat16, device="cuda")
    out = torch.empty_like(q)

    def attend(**change):
        a = dict(q=q, k_codes=cache[0], v_codes=cache[1], k_scale=cache[2], v_scale=cache[3], block_table=table, cu_q=ints([0, 1]), ctx_after=ints([40]),
                 out=out, max_q_len=1, num_heads=4, num_kv_heads=2, head_dim=64, block_size=16, scale=0.125, window=0,
                 scratch=torch.empty(1 << 20, dtype=torch.uint8, device="cuda"))
        a.update(change)
        k.attention_kv4(**a)

    attend()
    for match, change in (("heads must be a positive multiple", dict(num_heads=5, q=torch.zeros(1, 320, dtype=torch.bfloat16, device="cuda"), out=torch.zeros(1, 320, dtype=torch.bfloat16, device="cuda"))),
                          ("k_codes and v_codes must be", dict(k_codes=cache[2])), ("v_scale must be torch.uint8", dict(v_scale=cache[3].float())),
                          ("one length, one offset pair", dict(cu_q=ints([0, 1, 1]))), ("q and out must be", dict(out=out[:, :128].contiguous())),
                          ("a window must not be negative", dict(window=-1)), ("must be torch.bfloat16", dict(q=q.float())),
                          ("must be contiguous", dict(block_table=torch.cat([table, table], dim=1)[:, ::2])), ("CUDA tensor", dict(q=q.cpu()))):
        with pytest.raises(KernelError, match=match):
            attend(**change)
    long_table = torch.zeros(1, 2000, dtype=torch.int32, device="cuda")     # (sizes alone decide: this table could hold 32,000 positions)
    for scratch in (torch.empty(8, dtype=torch.uint8, device="cuda"), None):
        with pytest.raises(KernelError, match="bytes of scratch are needed"):
            attend(block_table=long_table, scratch=scratch)
    qkv = torch.zeros(1, 8 * 64, device="cuda")
    with pytest.raises(KernelError, match="width does not match"):
        k.append_kv4(qkv[:, :256].contiguous(), None, ints([0]), ints([0]), table, out, *cache, 4, 2, 64, 16)
    with pytest.raises(KernelError, match="one query row"):
        k.append_kv4(qkv, None, ints([0, 1]), ints([0]), table, out, *cache, 4, 2, 64, 16)
    blocks = torch.empty(3, 2, 16, 64, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(KernelError, match="positions to keep"):
        k.unpack_kv4(*cache, table, ints([40]), blocks, blocks.clone(), torch.empty_like(table), 2, 64, 16, -1)
    with pytest.raises(KernelError, match="results must be"):
        k.unpack_kv4(*cache, table, ints([40]), blocks, blocks[:2].contiguous(), torch.empty_like(table), 2, 64, 16)


# ---- sequences of one call ----------------------------------------------------------------------------------------------

def windowed_prompts(dim, block, before, new, window, heads=4, kv=2):
    """Prompts of unequal length and what run_step wants of them; ``oldest``: the first position that each sequence's queries see."""
    lengths = [b + n for b, n in zip(before, new)]
    cache, table = make_cache(kv, dim, block, lengths)
    cu = [0]
    for c in new:
        cu.append(cu[-1] + c)
    q = torch.randn(cu[-1], heads * dim, device="cuda").bfloat16()
    return cache, table, cu, lengths, [max(0, b - window + 1) for b in before], q


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("block", [16, 32, 64])
def test_what_is_not_finite_stays_in_its_sequence(monkeypatch, dim, block):
    """Prompts with a window: the prompt kernel's tiles of 64 keys begin and end outside of the blocks that a sequence's queries see.  A first sequence
    of nothing but NaN, blocks behind a window that others have taken since, and positions that have left it: none reaches another result."""
    take(monkeypatch, False)
    heads, kv, window, before, new = 4, 2, 100, [500, 530, 37, 300], [200, 130, 200, 1]
    cache, table, cu, lengths, oldest, q = windowed_prompts(dim, block, before, new, window)
    clean = run_step(lib(dim), q, cache, table, cu, lengths, heads, kv, dim, block, max(new), window)
    for s in range(4):
        mine = slice(cu[s], cu[s + 1])
        ref, sums, whole = plain_kv4.attention(q[mine].double().view(new[s], heads, dim), cached(cache, table, s, lengths[s], block, 0),
                                               cached(cache, table, s, lengths[s], block, 1), before[s], 1.0 / math.sqrt(dim), window)
        allowed = HALF_STEP * ref.abs() + (2.0 ** -8 + 2.0 ** -11) * sums + 2.0 ** -32 * whole
        assert bool(((clean[mine].double().view(new[s], heads, dim) - ref).abs() <= allowed).all()), s
    spoiled = [c.clone() for c in cache]
    for of in (2, 3):
        spoiled[of][table[0, :-(-lengths[0] // block)].long()] = plain_kv4.NOT_FINITE
        for s in (1, 2, 3):
            kept, inside = oldest[s] // block, oldest[s] % block
            spoiled[of][table[s, kept].long(), :, :inside] = plain_kv4.NOT_FINITE
    moved = table.clone()
    for s in (1, 2, 3):
        moved[s, :oldest[s] // block] = table[0, 0]
    got = run_step(lib(dim), q, spoiled, moved, cu, lengths, heads, kv, dim, block, max(new), window)
    assert bool(torch.isnan(got[:cu[1]]).all())
    assert torch.equal(got[cu[1]:], clean[cu[1]:])


@pytest.mark.parametrize("block", [16, 64])
@pytest.mark.parametrize("few", [False, True])
def test_entries_of_blocks_that_nobody_sees_are_not_read(monkeypatch, block, few):
    """Behind a window and behind a sequence's end a table may hold anything."""
    take(monkeypatch, few)
    heads, kv, dim, window, before, new = 4, 2, 64, 100, [500, 530, 37, 300], [200, 130, 200, 1]
    cache, table, cu, lengths, oldest, q = windowed_prompts(dim, block, before, new, window)
    clean = run_step(lib(dim), q, cache, table, cu, lengths, heads, kv, dim, block, max(new), window)
    for s in range(4):
        table[s, :oldest[s] // block] = -2 ** 31
        table[s, -(-lengths[s] // block):] = 2 ** 31 - 1
    assert torch.equal(run_step(lib(dim), q, cache, table, cu, lengths, heads, kv, dim, block, max(new), window), clean)


@pytest.mark.parametrize("window", [0, 150])
def test_prompts_read_back_in_pieces_without_new_tokens(monkeypatch, window):
    """Pieces all of whose sequences bring no token between pieces that bring some, one sequence at a time through one scratch: nobody's keys are
    written over while they are read."""
    from stratakv_b200 import ops
    k = lib(64)
    heads, kv, block, before, new = 8, 2, 64, [900, 2000, 2000, 40, 700, 2000, 300], [200, 0, 0, 200, 130, 0, 170]
    lengths = [b + n for b, n in zip(before, new)]
    cache, table = make_cache(kv, 64, block, lengths)
    cu = [0]
    for c in new:
        cu.append(cu[-1] + c)
    q = torch.randn(cu[-1], heads * 64, device="cuda").bfloat16()
    take(monkeypatch, False)
    whole = k.attention_kv4_scratch(7, cu[-1], 200, table.shape[1], heads, kv, 64, block, window)
    monkeypatch.setattr(ops, "KV4_UNPACKED", whole // 7)
    assert k.attention_kv4_scratch(7, cu[-1], 200, table.shape[1], heads, kv, 64, block, window) == whole // 7
    alone = {s: run_step(k, q[cu[s]:cu[s + 1]].contiguous(), cache, table[s:s + 1].contiguous(), [0, new[s]], [lengths[s]], heads, kv, 64, block, 200, window)
             for s in range(7) if new[s]}
    for _ in range(20):
        got = run_step(k, q, cache, table, cu, lengths, heads, kv, 64, block, 200, window)
        for s, result in alone.items():
            assert torch.equal(got[cu[s]:cu[s + 1]], result), s


@pytest.mark.parametrize("power", [10, 17, 24, 30, 120])
@pytest.mark.parametrize("dim,few", [(64, True), (128, True), (80, True), (64, False), (128, False)])
def test_queries_of_a_wide_range(monkeypatch, dim, few, power):
    """A number of a query head that is many times the others and meets zeros: what the others say decides.  A number of the head is off by at most
    2^-40 of the power of two below the largest, as a half's last place is 2^-24 and the largest is brought to 2^15."""
    take(monkeypatch, few)
    k = lib(dim)
    heads, kv, block, before, new = 4, 2, 16, [400, 90], [3, 2]
    lengths = [b + n for b, n in zip(before, new)]
    cache, table = make_cache(kv, dim, block, lengths, spread=3.0)
    cache[0][..., 0] = cache[0][..., 0] & 0xF0 | 8                # (number 0 of every key: 0)
    cu = [0, new[0], sum(new)]
    q = torch.randn(cu[-1], heads * dim, device="cuda").bfloat16()
    q[:, 0::dim] = 2.0 ** power * 1.9921875
    got = run_step(k, q, cache, table, cu, lengths, heads, kv, dim, block, max(new))
    for s in range(2):
        mine = slice(cu[s], cu[s + 1])
        keys = cached(cache, table, s, lengths[s], block, 0)
        rows = q[mine].double().view(new[s], heads, dim)
        if power > 50:                                            # (the others are below a half's last place)
            rows = torch.zeros_like(rows) if few else rows
        ref, sums, whole = plain_kv4.attention(rows, keys, cached(cache, table, s, lengths[s], block, 1), before[s], 1.0 / math.sqrt(dim))
        # scores off by d change weights by a factor of e^(2 d) at most
        off = 2.0 ** (power - 40) * float(keys.abs().sum(-1).max()) / math.sqrt(dim) if few and power < 50 else 0.0
        allowed = HALF_STEP * ref.abs() + ((2.0 ** -11 if few else 2.0 ** -8) + 2.0 ** -11 + math.expm1(2 * off)) * sums + 2.0 ** -32 * whole
        assert bool(((got[mine].double().view(new[s], heads, dim) - ref).abs() <= allowed).all()), (s, off)


@pytest.mark.parametrize("window", [0, 100])
@pytest.mark.parametrize("few", [False, True])
@pytest.mark.parametrize("block", [16, 64])
def test_a_length_beyond_the_table_is_cut(monkeypatch, block, few, window):
    """To the positions that the table has, whichever way a step takes."""
    take(monkeypatch, few)
    k = lib(64)
    heads, kv, before, new = 4, 2, [440, 300, 440], [200, 70, 200]      # (640 positions fill the table)
    lengths = [b + n for b, n in zip(before, new)]
    cache, table = make_cache(kv, 64, block, lengths)
    cu = [0, 200, 270, 470]
    q = torch.randn(470, heads * 64, device="cuda").bfloat16()
    clean = run_step(k, q, cache, table, cu, lengths, heads, kv, 64, block, 200, window)
    assert bool(torch.isfinite(clean).all())
    assert torch.equal(run_step(k, q, cache, table, cu, [641, 370, 10 ** 5], heads, kv, 64, block, 200, window), clean)


@pytest.mark.parametrize("new", [1, 200])
@pytest.mark.parametrize("scale", [0.0, -0.125, math.nan, math.inf])
def test_a_scale_that_is_not_positive_is_refused(monkeypatch, new, scale):
    """Prompts mask a score by minus infinity ahead of the scale."""
    from stratakv_b200.ops import KernelError
    take(monkeypatch, new == 1)
    k = lib(64)
    cache, table = make_cache(2, 64, 16, [300 + new])
    q = torch.randn(new, 4 * 64, device="cuda").bfloat16()
    out = torch.full_like(q, 7.0)
    scratch = torch.empty(k.attention_kv4_scratch(1, new, new, table.shape[1], 4, 2, 64, 16), dtype=torch.uint8, device="cuda")
    with pytest.raises(KernelError, match="scale must be positive"):
        k.attention_kv4(q, *cache, table, ints([0, new]), ints([300 + new]), out, new, 4, 2, 64, 16, scale, 0, scratch)
    assert bool((out == 7.0).all())


@pytest.mark.parametrize("heads,kv,block,before,new,window", [
    (6, 2, 64, [0], [1], 0), (6, 2, 16, [299, 16, 40], [1, 1, 1], 0), (16, 16, 32, [70, 500], [1, 1], 33), (24, 1, 64, [600], [3], 0), (4, 4, 48, [90, 0], [50, 7], 0),
    (8, 2, 32, [0, 77], [200, 130], 100), (6, 2, 64, [17000, 511], [1, 1], 0)])
def test_attention_of_heads_of_96(heads, kv, block, before, new, window):
    """(A key's 48 bytes of codes are three pieces, which no power of two of lanes shares out.)"""
    check_attention(heads, kv, 96, block, before, new, window)


def test_append_and_read_back_of_heads_of_96():
    from stratakv_b200.parts.position import rope_table
    heads, kv, dim, block, new = 5, 1, 96, 16, [33, 1, 20]
    k = lib(dim)
    cache, table = make_cache(kv, dim, block, new)
    n = sum(new)
    qkv = torch.randn(n, (heads + 2 * kv) * dim, device="cuda")
    positions = torch.cat([torch.arange(c) for c in new]).int().cuda()
    seqs = torch.repeat_interleave(torch.arange(3), torch.tensor(new)).int().cuda()
    cos_sin = torch.from_numpy(rope_table(dim, 10000.0, 40)).cuda()
    q_out = torch.empty(n, heads * dim, dtype=torch.bfloat16, device="cuda")
    k.append_kv4(qkv, cos_sin, positions, seqs, table, q_out, *cache, heads, kv, dim, block)
    rows = qkv.view(n, heads + 2 * kv, dim)
    turned = plain_kv4.rotate(rows[:, :heads + kv], cos_sin, positions)
    assert torch.equal(q_out, turned[:, :heads].flatten(1).bfloat16())
    out = [torch.empty(table.numel(), kv, block, dim, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    k.unpack_kv4(*cache, table, ints(new), *out, torch.empty_like(table), kv, dim, block)
    for of, x in ((0, turned[:, heads:]), (1, rows[:, heads + kv:])):
        plain = plain_kv4.read(*plain_kv4.store(x))
        got = out[of].view(3, table.shape[1], kv, block, dim).transpose(1, 2).flatten(2, 3)
        for s, c in enumerate(new):
            assert torch.equal(got[s, :, :c].double(), plain[seqs == s].transpose(0, 1)) and bool((got[s, :, c:] == 0).all())


@pytest.mark.parametrize("few", [False, True])
def test_a_step_without_any_token(monkeypatch, few):
    """Sequences, but no rows: nothing to do, whichever way the sizes would take."""
    take(monkeypatch, few)
    cache, table = make_cache(2, 64, 64, [300, 40])
    q = torch.empty(0, 4 * 64, device="cuda", dtype=torch.bfloat16)
    assert run_step(lib(64), q, cache, table, [0, 0, 0], [300, 40], 4, 2, 64, 64, 200).shape == (0, 256)
