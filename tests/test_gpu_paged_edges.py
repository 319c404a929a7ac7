"""GPU tests of the paged cache's operators (cactus_amd/paged.py) where numbers are small, infinite or not numbers: weights far
below the largest, infinite values that are seen, page scales that no append makes, codes that are requantized many times."""
import math

import pytest

from tests import paged_reference as R
from tests.test_gpu_paged import check_append, check_attention, random_cache, read_back

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def P():
    import cactus_amd.hip as hip
    import cactus_amd.paged as paged
    hip.init(0)
    return paged


def i32(x):
    return torch.tensor(x, dtype=torch.int32)


# ------------------------------------------------------------------------------------- weights far below the largest

# A weight is rounded to binary16 after it was raised by 2^11 against a maximum that is at most 2^4 behind, so it is off by half a
# step, 2^-11 of itself, or 2^-25 of the raised unit: 2^-36 of the largest weight.
SMALLEST = 2.0 ** -36


def first_key_and_the_rest(bits, keys):
    """exp2 weights: 1 for key 0, whose value is zero, and 2^-bits for each of the others, whose values are one."""
    w = 2.0 ** -bits
    total = 1 + (keys - 1) * w
    want = (keys - 1) * w / total
    # the weights' rounding; scores (one product of small numbers each) and their base-2 argument in fp32: 4 roundings of `bits`; the
    # sums' over the keys; the output's own
    tol = (keys - 1) * (max(w * R.U16, SMALLEST) + w * (4 * bits * R.U32 + keys * R.U32)) / total + want * R.U16 + 2.0 ** -25
    return want, tol


@pytest.mark.parametrize("bits", [10, 14.25, 17.5, 20, 21.75, 23.5, 24.5, 25.25, 26.5])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_many_small_weights_beside_a_large_one(P, D, bits):
    """What a first token without a value of its own does: it takes nearly all of the weight and the others share the rest."""
    n, page, scale = 8192, 64, math.log(2)
    want, tol = first_key_and_the_rest(bits, n)
    q, k, v = (torch.zeros((n, 1, D), dtype=torch.float16, device="cuda") for _ in range(3))
    q[:, 0, 0] = 1.0
    k[0, 0, 0] = bits
    v[1:] = 1.0
    out = P.attention_ragged(q, k, v, i32([0, n]).cuda(), scale=scale)[-1].cpu().double()
    assert bool(((out - want).abs() <= tol).all()), float(out[0, 0] / want - 1)
    kv = P.empty_pages(n // page, 1, D, page)
    kv[0].view(-1, D)[0, 0] = int(4 * bits)
    kv[1].view(-1, D)[1:] = 64
    kv[2].fill_(0.25)
    kv[3].fill_(1 / 64)
    t = torch.arange(n // page, dtype=torch.int32, device="cuda")[None]
    one = P.attention(q[:1], kv, t, i32([n]).cuda(), scale=scale)[-1].cpu().double()
    many = P.attention(q[:70], kv, t, i32([n]).cuda(), cu_seqlens=i32([0, 70]).cuda(), scale=scale)[-1].cpu().double()
    # over pages the weights of a launch's key splits are raised against each split's own maximum, which only helps
    assert bool(((one - want).abs() <= tol).all()), float(one[0, 0] / want - 1)
    assert bool(((many - want).abs() <= tol).all()), float(many[0, 0] / want - 1)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("step", [0.5, 3.0, 5.0])
def test_a_maximum_that_grows_with_every_key(P, D, step):
    """Scores that rise from key to key: the running maximum moves all the time, by less and by more than it may be behind."""
    n, page, scale = 700, 16, math.log(2)
    top = 127 * 0.25                                     # of the scores, as codes of scale 1/4 can hold them
    codes = torch.arange(n).float().mul(4 * step).sub(4 * step * (n - 1)).add(4 * top).clamp_min(-508).div(4).round()
    k = torch.zeros((n, 1, D), dtype=torch.float16)
    k[:, 0, 0] = codes * 0.25
    v = torch.randint(-127, 128, (n, 1, D), generator=torch.Generator().manual_seed(D)).half() / 64
    q = torch.zeros((n, 1, D), dtype=torch.float16)
    q[:, 0, 0] = 4.0
    rows = torch.tensor([0, 1, 15, 16, 63, 64, 65, 300, 511, n - 1])
    want, tol = R.attend(q[rows], k, v, rows, 0, 0, scale)
    out = P.attention_ragged(q.cuda(), k.cuda(), v.cuda(), i32([0, n]).cuda(), scale=scale).cpu().double()
    assert bool(((out[rows] - want).abs() <= tol).all())
    kv = [x.cuda() for x in P.empty_pages((n + page - 1) // page, 1, D, page)]
    flat = lambda x: torch.cat([x[:, 0], x.new_zeros((-n % page, D))]).view(-1, 1, page, D).to(torch.int8).cuda()  # noqa: E731
    kv[0].copy_(flat(k.float() * 4))
    kv[1].copy_(flat(v.float() * 64))
    kv[2].fill_(0.25)
    kv[3].fill_(1 / 64)
    t = torch.arange(kv[0].shape[0], dtype=torch.int32, device="cuda")[None]
    for m in (1, 60):
        cu = None if m == 1 else i32([0, m]).cuda()
        got = P.attention(q[:m].cuda(), kv, t, i32([n]).cuda(), cu_seqlens=cu, scale=scale)[-1:].cpu().double()
        assert bool(((got - want[-1:]).abs() <= tol[-1:]).all()), m


# ------------------------------------------------------------------------------------------- infinite values that are seen

def check_infinities(P, D, H, lengths, window, sink, rows, heads):
    """Values that are not finite in tiles that rows see whole and in those they do not, on keys that weigh next to nothing (about
    2^-46 at head_dim 64, 2^-92 at 256) beside the first key of a sequence, or beside a later one that outgrows what came before."""
    gen = torch.Generator().manual_seed(D + window)
    T, n, base = sum(lengths), lengths[-1], sum(lengths[:-1])
    q = torch.ones((T, H, D), dtype=torch.float16)
    k = (torch.randn((T, H, D), generator=gen) / 16).half()
    v = torch.randn((T, H, D), generator=gen).half()
    k[base] = 4.0
    k[base + n // 2] = 8.0
    for key, dim, x in ((1, 0, math.inf), (20, 7, math.inf), (33, 7, math.inf), (70, 8, -math.inf), (5, 9, math.inf), (140, 9, -math.inf),
                        (64, D - 1, math.nan), (n - 40, 40, -math.inf), (n - 1, 41, math.inf), (n - 2, 42, math.nan)):
        v[base + key, :, dim] = x
    cu = R.offsets(lengths)
    out = P.attention_ragged(q.cuda(), k.cuda(), v.cuda(), cu.cuda(), window=window, sink=sink).cpu().double()
    assert bool(torch.isfinite(out[:base]).all())
    at = torch.tensor(rows)
    for h in heads:
        one = slice(h, h + 1)
        want, tol = R.attend(q[base + at, one], k[base:, one], v[base:, one], at, window, sink)
        got, fine = out[base + at, one], torch.isfinite(want)
        assert not bool(fine.all())
        assert bool((torch.isnan(got) == torch.isnan(want)).all())
        whole = ~torch.isnan(want) & ~fine
        assert bool((got[whole] == want[whole]).all())
        assert bool(((got - want).abs() <= tol)[fine].all())


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("window,sink", [(0, 0), (90, 0), (100, 6), (150, 70)])
def test_infinite_values_on_keys_of_no_weight(P, D, window, sink):
    n = 330
    rows = [0, 1, 5, 19, 20, 21, 33, 63, 64, 69, 70, 100, 110, 127, 128, 140, 141, 164, 165, 166, 200, 255, 256, 289, 290, 291, 328, 329]
    check_infinities(P, D, 2, [37, n], window, sink, rows, [0, 1])


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("window,sink", [(0, 0), (300, 6)])
def test_infinite_values_where_one_group_takes_all_keys(P, D, window, sink):
    check_infinities(P, D, 40, [300, 1400], window, sink, [0, 20, 69, 140, 320, 321, 641, 699, 700, 1000, 1359, 1360, 1399], [0, 39])


@pytest.mark.parametrize("D", [64, 128, 256])
def test_infinite_values_behind_a_query_that_is_not_a_number(P, D):
    """The row of such a query is not a number in any dim, its neighbours are what they would be without it."""
    gen = torch.Generator().manual_seed(D)
    n = 200
    q, k, v = (torch.randn((n, 1, D), generator=gen).half().cuda() for _ in range(3))
    v[3, 0, 5] = math.inf
    want = P.attention_ragged(q, k, v, i32([0, n]).cuda())
    q[150, 0, 9] = math.nan
    got = P.attention_ragged(q, k, v, i32([0, n]).cuda())
    assert bool(torch.isnan(got[150]).all())
    want[150] = got[150] = 0
    assert torch.equal(got, want) and bool((got[3:150, 0, 5] == math.inf).all()) and bool(torch.isfinite(got[:3]).all())


# ------------------------------------------------------------------------------------------- page scales that are none

@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("bad", [-0.02, -0.0, math.nan, math.inf, -math.inf])
def test_a_scale_that_is_not_positive_and_finite_counts_as_zero(P, D, which, bad):
    """In every call alike: one row, many rows, tokens read back, tokens appended behind such ones."""
    gen = torch.Generator().manual_seed(D)
    page, H, n = 16, 2, 75
    kv = [torch.randint(-127, 128, (5, H, page, D), generator=gen, dtype=torch.int8).cuda() for _ in range(2)]
    kv += [(0.01 + 0.02 * torch.rand((5, H), generator=gen)).cuda() for _ in range(2)]
    q = torch.randn((40, 4, D), generator=gen).half().cuda()
    rows = torch.randn((3, H, D), generator=gen).half().cuda()
    t, ctx = i32([[3, 1, 0, 2, 4]]).cuda(), i32([n]).cuda()

    def results(value):
        x = [y.clone() for y in kv]
        x[2 if which == "k" else 3][[1, 4]] = value
        out = [P.attention(q[39:], x, t, ctx), P.attention(q, x, t, ctx, cu_seqlens=i32([0, 40]).cuda()),
               P.attention(q[:3], x, t, ctx, cu_seqlens=i32([0, 3]).cuda())]
        out += P.kv_read(x, t, i32([0]).cuda(), i32([0, n]).cuda(), n)
        P.kv_append(rows, rows, x, t, i32([n]).cuda(), 1e4, cu_seqlens=i32([0, 3]).cuda())
        return out + [y[4] for y in x]

    for a, b in zip(results(bad), results(0.0)):
        assert bool(torch.isfinite(a).all()) and bool((a == b).all())


# ------------------------------------------------------------------------------------------- hints, many pages, many sequences

@pytest.mark.parametrize("D,page", [(64, 16), (128, 32), (256, 64)])
@pytest.mark.parametrize("window,sink", [(0, 0), (300, 4)])
def test_the_bound_of_a_chunk_batch_is_only_a_hint(P, D, page, window, sink):
    for hint in (0, 127, 1 << 30):
        check_attention(P, 3, D, page, 4, 2, [70, 0, 130, 1], [900, 3, 1301, 40], window, sink, max_context=hint)


# How the launch cuts an append: workgroups for 1024 (page, items) pieces, all items of a page in one where there are as many
# pages.  Pieces are floor(tokens / page) + 2 * sequences, at one row each one a sequence; a pass of a workgroup takes 256 or more
# row slots of D / 16 lanes, so several items or query heads more than fit one need more passes.

@pytest.mark.parametrize("D,page,Hq,Hkv,sequences", [(64, 16, 9, 3, 500), (64, 32, 6, 3, 520), (64, 64, 4, 2, 520), (128, 16, 3, 3, 500),
                                                     (128, 64, 4, 2, 520), (256, 16, 2, 2, 500), (256, 128, 3, 1, 520)])
def test_append_of_many_pages_in_several_passes(P, D, page, Hq, Hkv, sequences):
    gen = torch.Generator().manual_seed(D + page)
    news = [int(x) for x in torch.randint(0, 24, (sequences,), generator=gen)]
    pasts = [int(x) for x in torch.randint(0, 3 * page, (sequences,), generator=gen)]
    for b, n in ((0, 3 * page + 1), (70, 0), (200, 2 * page), (sequences - 1, page + 3)):
        news[b] = n
    pasts[300], pasts[301] = -1, -5
    pieces = sum(news) // page + 2 * sequences
    lanes = D // 16
    slots = max(256, page * lanes if page * lanes <= 256 else page * lanes // 2) // lanes
    assert pieces >= 1024 and 2 * Hkv > slots // min(page, slots) and Hq > slots // min(page, slots) // 2
    check_append(P, 21, D, page, Hq, Hkv, news, pasts)


@pytest.mark.parametrize("D,Hq,Hkv", [(64, 80, 40), (128, 40, 20), (256, 18, 9)])
def test_append_of_many_sequences_in_several_passes(P, D, Hq, Hkv):
    gen = torch.Generator().manual_seed(D)
    assert 2 * Hkv > 256 // (D // 16) and Hq > 256 // (D // 16)
    pasts = [int(x) for x in torch.randint(0, 40, (1030,), generator=gen)]
    pasts[3], pasts[1029] = -1, 16
    check_append(P, 22, D, 16, Hq, Hkv, [1] * 1030, pasts, use_cu=False)


def test_append_of_long_prompts_in_several_passes(P):
    news, pasts = [1203, 1187, 1250, 1100, 1333, 1211, 1197], [0, 5, 31, 32, 33, 700, 0]
    check_append(P, 23, 64, 32, 32, 8, news, pasts)


@pytest.mark.parametrize("sequences", [64, 65, 66, 130, 200, 1000])
def test_append_and_read_of_many_sequences(P, sequences):
    """More sequences than a wave looks through at once, some of them without rows."""
    gen = torch.Generator().manual_seed(sequences)
    D, page, Hkv = 64, 16, 2
    news = [int(x) for x in torch.randint(0, 5, (sequences,), generator=gen)]
    pasts = [int(x) for x in torch.randint(0, 40, (sequences,), generator=gen)]
    news[0], news[sequences // 2], news[sequences - 1] = 0, 50, 0
    check_append(P, 24, D, page, 4, Hkv, news, pasts)
    starts = [int(x) for x in torch.randint(0, 30, (sequences,), generator=gen)]
    used = [(c + s + page - 1) // page for c, s in zip(news, starts)]
    total = sum(used) + 2
    tables = R.make_tables(gen, used, max(used), total)
    kv = random_cache(gen, total, Hkv, page, D)
    k, v = P.kv_read([x.cuda() for x in kv], tables.cuda(), i32(starts).cuda(), R.offsets(news).cuda(), sum(news))
    want = [torch.cat([R.gather(x, y, tables[b], page, s, c)[0] for b, (c, s) in enumerate(zip(news, starts))])
            for x, y in ((kv[0], kv[2]), (kv[1], kv[3]))]
    assert read_back(k, want[0]) and read_back(v, want[1])


# ------------------------------------------------------------------------------------------- codes requantized many times

@pytest.mark.parametrize("page", [16, 64, 128])
@pytest.mark.parametrize("growth", ["normal", "spread", "slow"])
def test_token_by_token_a_code_is_off_by_half_of_every_scale_it_had(P, page, growth):
    """The cache against the FP16 rows themselves, over two pages filled a token at a time and in calls of five.  Each time a page's
    scale grows its codes are rounded once more, by at most half a step of the new scale."""
    gen = torch.Generator().manual_seed(page)
    D, H, n = 128, 2, 2 * page
    x = torch.randn((n, 2, H, D), generator=gen).clamp(-2.5, 2.5)
    at = torch.arange(n).float().view(-1, 1, 1, 1)
    x *= {"normal": 1 + 0 * at, "spread": torch.exp(0.5 * torch.randn((n, 1, 1, 1), generator=gen)), "slow": 1.004 ** at}[growth]
    x = x.half()
    t = i32([[1, 0]])
    for step in (1, 5):
        kv = P.empty_pages(2, H, D, page)
        scales, bound = torch.zeros((2, 2, H), dtype=torch.float64), torch.zeros((2, 2, H), dtype=torch.float64)
        for i in range(0, n, step):
            m = min(step, n - i)
            rows = x[i:i + m].cuda()
            P.kv_append(rows[:, 0], rows[:, 1], kv, t.cuda(), i32([i]).cuda(), 0.0, cu_seqlens=i32([0, m]).cuda())
            now = torch.stack([kv[2].cpu(), kv[3].cpu()]).double()
            bound += torch.where(now > scales, 0.5 * now * (1 + 2 * 127 * 4 * R.U32), 0.0)
            scales = now
        back = [R.gather(kv[w].cpu(), kv[2 + w].cpu(), t[0], page, 0, n)[0] for w in range(2)]
        for w in range(2):
            for p in range(2):
                err = (back[w][p * page:(p + 1) * page] - x[p * page:(p + 1) * page, w].double()).abs()
                assert bool((err.amax((0, 2)) <= bound[w, int(t[0, p])]).all())


# ------------------------------------------------------------------------------------------- results in place of the queries

@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("news,contexts", [([1] * 5, [1, 700, 64, 0, 300]), ([1], [5000]), ([70, 1, 0, 130], [900, 40, 3, 1301]), ([150], [150]),
                                           ([3, 2, 40], [1000, 2, 2000])])
def test_outputs_may_be_the_queries(P, D, news, contexts):
    gen = torch.Generator().manual_seed(D)
    page, Hq, Hkv, T = 32, 6, 2, sum(news)
    used = [(c + page - 1) // page for c in contexts]
    kv = [x.cuda() for x in random_cache(gen, sum(used) + 1, Hkv, page, D)]
    t = R.make_tables(gen, used, max(used), sum(used) + 1).cuda()
    cu = R.offsets(news).cuda()
    ctx = i32(contexts).cuda()
    q, k, v = (torch.randn((T, h, D), generator=gen).half().cuda() for h in (Hq, Hkv, Hkv))
    past = ctx - (cu[1:] - cu[:-1])
    calls = [lambda x, out: P.attention(x, kv, t, ctx, cu_seqlens=None if max(news) == 1 else cu, out=out),
             lambda x, out: P.attention_ragged(x, k, v, cu, window=50, sink=3, out=out),
             lambda x, out: P.kv_append(k, v, [y.clone() for y in kv], t, past, 1e4, cu_seqlens=cu, q=x, out_q=out)]
    for call in calls:
        own = q.clone()
        want = call(q, q.clone())        # rows of a sequence that is skipped (a context of 0: position -1) stay as they were
        assert call(own, own) is own
        assert torch.equal(own, want)
