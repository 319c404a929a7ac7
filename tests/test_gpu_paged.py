"""GPU tests of the paged INT8 cache (cactus_amd/paged.py) against tests/paged_reference.py: append with norm, rotation and
page scales, read-back, attention over the pages, ragged prompt attention, and all of them in a row."""
import math

import pytest

from tests import paged_reference as R

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def P():
    import cactus_amd.hip as hip
    import cactus_amd.paged as paged
    hip.init(0)
    return paged


def gpu(*xs):
    out = [x.cuda() for x in xs]
    return out[0] if len(out) == 1 else out


def i32(x):
    return torch.tensor(x, dtype=torch.int32)


def random_cache(gen, pages, heads, page, D):
    mk = lambda: torch.randint(-127, 128, (pages, heads, page, D), generator=gen, dtype=torch.int8)  # noqa: E731
    sc = lambda: 0.005 + 0.03 * torch.rand((pages, heads), generator=gen)  # noqa: E731
    return mk(), mk(), sc(), sc()


# ------------------------------------------------------------------------------------------------------------- append

def check_append(P, seed, D, page, Hq, Hkv, news, pasts, theta=1e6, norm=True, use_cu=True, fused=True, width=None, edit=None,
                 with_q=True, spoil=None):
    """Runs the call and compares every byte of the cache and every row of q.  edit(tables): changes to the block tables;
    spoil(k, v): changes to the inputs."""
    gen = torch.Generator().manual_seed(seed)
    T, eps = sum(news), 1e-6
    used = [(max(p, 0) + n + page - 1) // page for n, p in zip(news, pasts)]
    if width:
        used = [min(u, width) for u in used]
    total = sum(used) + 2
    tables = R.make_tables(gen, used, width or max(used) + 1, total)
    if edit:
        edit(tables)
    kv = random_cache(gen, total, Hkv, page, D)
    rows = torch.randn((T, (Hq + 2 * Hkv) * D), generator=gen).half()
    if spoil:
        spoil(rows.view(T, Hq + 2 * Hkv, D))
    q, k, v = (rows[:, a * D:b * D].unflatten(1, (b - a, D)) for a, b in ((0, Hq), (Hq, Hq + Hkv), (Hq + Hkv, Hq + 2 * Hkv)))
    qw, kw = ((1 + 0.2 * torch.randn(D, generator=gen)).half() for _ in range(2))
    cu = R.offsets(news)
    dev = [x.clone().cuda() for x in kv]
    rows_d = rows.cuda()
    qd, kd, vd = (rows_d[:, a * D:b * D].unflatten(1, (b - a, D)) for a, b in ((0, Hq), (Hq, Hq + Hkv), (Hq + Hkv, Hq + 2 * Hkv)))
    if not fused:
        qd, kd, vd = qd.contiguous(), kd.contiguous(), vd.contiguous()
    out = torch.full((T, Hq, D), 7.0, dtype=torch.float16, device="cuda") if with_q else None
    got = P.kv_append(kd, vd, dev, tables.cuda(), i32(pasts).cuda(), theta, cu_seqlens=cu.cuda() if use_cu else None,
                      q=qd if with_q else None, q_weight=qw.cuda() if norm else None, k_weight=kw.cuda() if norm else None,
                      eps=eps, out_q=out)
    torch.cuda.synchronize()
    assert got is out
    new = [x.cpu() for x in dev]
    same = torch.ones(total, dtype=torch.bool)      # pages that keep every byte
    rel = R.row_bound(D)
    for b, (n, p) in enumerate(zip(news, pasts)):
        r = slice(int(cu[b]), int(cu[b]) + n)
        if p < 0:
            if with_q:
                assert bool((got[r] == 7.0).all())
            continue
        pos = torch.arange(p, p + n)
        if with_q:
            want, terms = R.norm_rope(q[r], qw if norm else None, eps, theta, pos)
            tol = R.U16 * want.abs() + terms * rel + 2.0 ** -24
            ok = torch.isfinite(want) & (want.abs() < 65000)
            assert bool(((got[r].cpu().double() - want).abs() <= tol)[ok].all())
        kk = R.norm_rope(R.finite(k[r]), kw if norm else None, eps, theta, pos)
        vv = (R.finite(v[r]), R.finite(v[r]).abs())
        for j in range(p // page, (p + n + page - 1) // page):
            lo, hi = max(p, j * page), min(p + n, (j + 1) * page)
            if hi <= lo or j >= tables.shape[1] or not 0 <= int(tables[b, j]) < total:
                continue
            pid = int(tables[b, j])
            same[pid] = False
            for (x, terms), before, after, s0, s1 in ((kk, kv[0], new[0], kv[2], new[2]), (vv, kv[1], new[1], kv[3], new[3])):
                x, terms = x[lo - p:hi - p].transpose(0, 1), terms[lo - p:hi - p].transpose(0, 1)
                held = lo - j * page
                old = s0[pid].double() if held else torch.zeros(Hkv, dtype=torch.float64)
                scale = torch.maximum(old, x.abs().amax((1, 2)) / 127).clamp_min(1e-10)
                off = rel * terms.amax((1, 2)) / 127 + 4 * R.U32 * scale
                assert bool(((s1[pid].double() - scale).abs() <= off).all())
                # a code is the value over the stored scale, rounded; a value may sit on the border of two codes
                y = x / s1[pid].double()[:, None, None]
                slack = 0.5 + rel * terms / s1[pid].double()[:, None, None] + 127 * 8 * R.U32
                assert bool(((after[pid, :, held:hi - j * page].double() - y).abs() <= slack).all())
                if held:
                    f = torch.where(s1[pid] > s0[pid], s0[pid].double() / s1[pid].double(), torch.ones(Hkv, dtype=torch.float64))
                    moved = before[pid, :, :held].double() * f[:, None, None]
                    assert bool(((after[pid, :, :held].double() - moved).abs() <= 0.5 + 127 * 4 * R.U32).all())
                    kept = f == 1
                    assert torch.equal(after[pid, kept, :held], before[pid, kept, :held])
                assert torch.equal(after[pid, :, hi - j * page:], before[pid, :, hi - j * page:])
    for before, after in zip(kv, new):
        assert torch.equal(before[same], after[same])


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
def test_append_one_row_each(P, D, page):
    pasts = [0, 1, page - 1, page, page + 1, 3 * page - 1, 3 * page, 700]
    check_append(P, D + page, D, page, 4, 2, [1] * len(pasts), pasts, use_cu=False)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
def test_append_ragged(P, D, page):
    news = [page, 1, 0, page + 1, 2 * page - 1, 3, 5 * page + 7]
    pasts = [0, page - 1, 5, page // 2, 2 * page + 1, 0, page - 3]
    check_append(P, 3 * D + page, D, page, 6, 2, news, pasts, theta=1e4)


@pytest.mark.parametrize("Hq,Hkv", [(16, 8), (32, 8), (4, 1), (9, 3), (1, 1), (40, 40), (300, 100)])
@pytest.mark.parametrize("use_cu", [False, True])
def test_append_heads(P, Hq, Hkv, use_cu):
    check_append(P, Hq, 64, 16, Hq, Hkv, [1, 1, 1], [0, 17, 46], use_cu=use_cu)


@pytest.mark.parametrize("theta,norm,with_q,fused", [(0.0, False, True, True), (0.0, True, False, True), (1e4, False, True, False),
                                                     (1e6, True, True, False), (5e5, False, False, False)])
def test_append_options(P, theta, norm, with_q, fused):
    check_append(P, 11, 128, 32, 8, 4, [1, 40, 33], [100, 31, 0], theta=theta, norm=norm, with_q=with_q, fused=fused)
    check_append(P, 12, 128, 32, 8, 4, [1, 1], [100, 31], theta=theta, norm=norm, with_q=with_q, fused=fused, use_cu=False)


def test_append_at_far_positions(P):
    # an fp32 angle would be off by 2^-24 * 1e6 rad here
    check_append(P, 5, 128, 128, 4, 2, [3, 1], [1000003, 262143], theta=1e4)


@pytest.mark.parametrize("use_cu", [False, True])
def test_append_skips_what_has_no_place(P, use_cu):
    def edit(t):
        t[1, 0] = -1
        t[2, 1] = 1 << 30
        t[3, 0] = 1000
    check_append(P, 6, 64, 16, 4, 2, [1] * 6, [-1, 3, 16, 2, 40, -7], use_cu=use_cu, edit=edit)
    # past the end of the table
    check_append(P, 7, 64, 16, 4, 2, [1] * 3, [31, 32, 1 << 30] if use_cu else [31, 33, 48], use_cu=use_cu, width=2)


def test_append_stores_no_infinity(P):
    def spoil(rows):
        rows[0, 4, 3] = math.inf
        rows[0, 4, 9] = -math.inf
        rows[1, 5, 0] = math.nan
        rows[2, 6, 63] = math.nan
        rows[3, 7, :] = math.inf
        rows[4, 6, :] = 0
    check_append(P, 8, 64, 16, 4, 2, [1] * 5, [0, 5, 16, 31, 8], norm=False, use_cu=False, spoil=spoil)
    check_append(P, 9, 64, 16, 4, 2, [3, 2], [0, 5], norm=False, spoil=spoil)


def test_append_of_zero_rows_has_the_smallest_scale(P):
    kv = list(P.empty_pages(2, 1, 64, 16))
    z = torch.zeros((1, 1, 64), dtype=torch.float16, device="cuda")
    P.kv_append(z, z, kv, i32([[1]]).cuda(), i32([0]).cuda(), 1e4)
    assert kv[2].tolist()[1] == [pytest.approx(1e-10)] and kv[3].tolist()[0] == [0.0]
    assert not bool(kv[0].any())


def test_append_twice_changes_nothing(P):
    gen = torch.Generator().manual_seed(4)
    kv = [x.cuda() for x in random_cache(gen, 12, 2, 32, 64)]
    k, v = (torch.randn((50, 2, 64), generator=gen).half().cuda() * 3 for _ in range(2))
    args = (R.make_tables(gen, [3, 2], 3, 12).cuda(), i32([40, 7]).cuda(), 1e6)
    cu = R.offsets([30, 20]).cuda()
    P.kv_append(k, v, kv, *args, cu_seqlens=cu)
    once = [x.clone() for x in kv]
    P.kv_append(k, v, kv, *args, cu_seqlens=cu)
    assert all(torch.equal(a, b) for a, b in zip(once, kv))


def test_rows_behind_the_last_sequence_stay(P):
    gen = torch.Generator().manual_seed(4)
    kv = [x.cuda() for x in random_cache(gen, 12, 2, 16, 64)]
    before = [x.clone() for x in kv]
    rows = torch.randn((40, 2, 64), generator=gen).half().cuda()
    tables = R.make_tables(gen, [2, 1], 2, 12)
    out = torch.full((40, 2, 64), 7.0, dtype=torch.float16, device="cuda")
    cu = i32([0, 20, 23]).cuda()
    P.kv_append(rows, rows, kv, tables.cuda(), i32([0, 0]).cuda(), 1e4, cu_seqlens=cu, q=rows, out_q=out)
    assert bool((out[23:] == 7).all()) and not bool((out[:23] == 7).all())
    mine = torch.zeros(12, dtype=torch.bool)
    mine[tables[tables >= 0].long()] = True
    assert all(torch.equal(a.cpu()[~mine], b.cpu()[~mine]) for a, b in zip(before, kv))
    o2 = torch.full_like(out, 7.0)
    P.attention(out, kv, tables.cuda(), i32([20, 3]).cuda(), cu_seqlens=cu, out=o2)
    assert bool((o2[23:] == 7).all()) and not bool((o2[:23] == 7).any(-1).all())
    o3 = torch.full_like(out, 7.0)
    P.attention_ragged(out, rows, rows, cu, out=o3)
    assert bool((o3[23:] == 7).all())
    k2, v2 = torch.full_like(out, 7.0), torch.full_like(out, 7.0)
    P.kv_read(kv, tables.cuda(), i32([0, 0]).cuda(), cu, 40, out_k=k2, out_v=v2)
    assert bool((k2[23:] == 7).all()) and bool((v2[23:] == 7).all())


# --------------------------------------------------------------------------------------------------------------- read

def read_back(got, want):
    """code * scale rounded to a half.  The product may be rounded to fp32 on the way (2^-24 of it, which can carry a value
    across the middle between two halves) or not at all: half a step of a half, 2^-25 below 2^-14, and that 2^-24."""
    return bool(((got.cpu().double() - want).abs() <= want.abs() * (R.U16 + R.U32) + 2.0 ** -25).all())


@pytest.mark.parametrize("D,Hkv,page", [(64, 8, 16), (128, 1, 64), (256, 3, 128), (64, 1, 32)])
def test_read(P, D, Hkv, page):
    gen = torch.Generator().manual_seed(D)
    counts, starts = [1, 0, page + 5, 3 * page, 2], [0, 4, page - 2, 0, 5 * page - 1]
    used = [(c + s + page - 1) // page for c, s in zip(counts, starts)]
    total = sum(used) + 2
    tables = R.make_tables(gen, used, max(used), total)
    tables[2, 1] = -5
    kv = random_cache(gen, total, Hkv, page, D)
    k, v = P.kv_read(gpu(*kv), tables.cuda(), i32(starts).cuda(), R.offsets(counts).cuda(), sum(counts))
    at = 0
    for b, (c, s) in enumerate(zip(counts, starts)):
        for got, x, y in ((k, kv[0], kv[2]), (v, kv[1], kv[3])):
            want, _ = R.gather(x, y, tables[b], page, s, c)
            assert read_back(got[at:at + c], want)
        at += c


# ---------------------------------------------------------------------------------------------------- paged attention

def spread(scales):
    """How far the scales of written pages lie apart."""
    s = scales[scales > 0]
    return float(s.max() / s.min()) if s.numel() else 1.0


def check_attention(P, seed, D, page, Hq, Hkv, news, contexts, window=0, sink=0, use_cu=True, scale=0.0, edit=None, width=None,
                    max_context=None, strided=False, qscale=1.5):
    gen = torch.Generator().manual_seed(seed)
    used = [(c + page - 1) // page for c in contexts]
    total = sum(used) + 2
    tables = R.make_tables(gen, used, width or max(max(used), 1), total)
    kv = random_cache(gen, total, Hkv, page, D)
    dev = [x.cuda() for x in kv]
    owned = torch.zeros(total, dtype=torch.bool)
    owned[tables[tables >= 0].long()] = True
    for s in dev[2:]:
        s[~owned.cuda()] = math.nan            # pages of nobody are never looked at
    if edit:
        edit(tables)
    T = sum(news)
    q = (torch.randn((T, Hq, D), generator=gen) * qscale).half()
    qd = q.cuda()
    if strided:
        wide = torch.zeros((T, Hq * D + 24), dtype=torch.float16, device="cuda")
        wide[:, 8:8 + Hq * D] = qd.reshape(T, Hq * D)
        qd = wide[:, 8:8 + Hq * D].unflatten(1, (Hq, D))
    cu = R.offsets(news)
    out = P.attention(qd, dev, tables.cuda(), i32(contexts).cuda(), cu_seqlens=cu.cuda() if use_cu else None,
                      max_context=max_context, scale=scale, window=window, sink=sink)
    torch.cuda.synchronize()
    worst = 0.0
    for b, (n, c) in enumerate(zip(news, contexts)):
        k, ok = R.gather(kv[0], kv[2], tables[b], page, 0, c)
        v, _ = R.gather(kv[1], kv[3], tables[b], page, 0, c)
        r = slice(int(cu[b]), int(cu[b]) + n)
        want, tol = R.attend(q[r], k, v, torch.arange(c - n, c), window, sink, scale, ok, spread(kv[3]))
        err = (out[r].cpu().double() - want).abs()
        assert bool((err <= tol).all()), (b, n, c, float((err / tol).max()))
        worst = max(worst, float((err / tol).max()) if err.numel() else 0.0)
    return worst


SHAPES = [(64, 16, 8, 2), (128, 16, 4, 2), (128, 64, 16, 8), (256, 32, 4, 1), (64, 128, 9, 3), (256, 128, 2, 2)]


@pytest.mark.parametrize("D,page,Hq,Hkv", SHAPES)
def test_decode_contexts(P, D, page, Hq, Hkv):
    contexts = [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 200, 0, 511]
    check_attention(P, D + page, D, page, Hq, Hkv, [1] * len(contexts), contexts, use_cu=False)


@pytest.mark.parametrize("D,page,Hq,Hkv", SHAPES)
@pytest.mark.parametrize("window,sink", [(1, 0), (16, 0), (33, 4), (64, 17), (100, 1), (7, 70), (1000, 4), (60, 200)])
def test_decode_window(P, D, page, Hq, Hkv, window, sink):
    contexts = [1, 5, 17, 34, 64, 100, 133, 300]
    check_attention(P, window, D, page, Hq, Hkv, [1] * len(contexts), contexts, window, sink, use_cu=False)


@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (2, 1), (3, 1), (7, 1), (16, 1), (17, 1), (40, 2), (64, 1), (12, 12), (64, 64)])
def test_decode_groups(P, Hq, Hkv):
    check_attention(P, Hq, 64, 16, Hq, Hkv, [1, 1], [77, 130], use_cu=False)
    check_attention(P, Hq, 128, 16, Hq, Hkv, [1, 3], [77, 130])


@pytest.mark.parametrize("D,page,Hq,Hkv,context", [(128, 16, 4, 2, 5003), (64, 64, 4, 1, 9001), (256, 32, 4, 1, 4099), (128, 128, 2, 2, 20000)])
@pytest.mark.parametrize("window,sink", [(0, 0), (1500, 4)])
def test_decode_long(P, D, page, Hq, Hkv, context, window, sink):
    # one long sequence is split over workgroups; short neighbours leave most of their splits empty
    check_attention(P, 1, D, page, Hq, Hkv, [1], [context], window, sink, use_cu=False)
    check_attention(P, 2, D, page, Hq, Hkv, [1, 1, 1], [3, context, 0], window, sink, use_cu=False)
    check_attention(P, 3, D, page, Hq, Hkv, [1, 0, 2], [context - 1, 3, 40], window, sink, width=(context + page - 1) // page + 9)


def test_decode_max_context_is_only_a_hint(P):
    for hint in (0, 1, 100, 3000, 1 << 30):
        check_attention(P, 3, 128, 16, 4, 2, [1, 1], [2000, 3], use_cu=False, max_context=hint)


@pytest.mark.parametrize("D,page,Hq,Hkv", SHAPES)
@pytest.mark.parametrize("window,sink", [(0, 0), (40, 0), (70, 5)])
def test_chunks(P, D, page, Hq, Hkv, window, sink):
    news = [1, 2, 0, 5, 17, 64, 70, 130]
    contexts = [40, 2, 9, 200, 17, 64, 333, 131]
    check_attention(P, D + window, D, page, Hq, Hkv, news, contexts, window, sink, strided=True)


@pytest.mark.parametrize("D,Hq,Hkv", [(128, 4, 2), (64, 3, 1), (256, 2, 1)])
def test_chunk_of_many_rows(P, D, Hq, Hkv):
    check_attention(P, 1, D, 16, Hq, Hkv, [257], [1900])
    check_attention(P, 2, D, 64, Hq, Hkv, [300, 129], [300, 1025], 200, 4)


def test_context_shorter_than_the_rows(P):
    # the first rows of such a call stand before position 0 and see nothing
    check_attention(P, 1, 64, 16, 2, 1, [4, 20], [2, 3])
    check_attention(P, 1, 64, 16, 2, 1, [1, 1], [0, 0], use_cu=False)


@pytest.mark.parametrize("news", [[1, 1, 1], [3, 1, 40]])
def test_pages_that_are_missing_are_not_seen(P, news):
    def edit(t):
        t[0, 1] = -1
        t[1, 0] = 1 << 30
        t[2, :] = -3
    check_attention(P, 1, 64, 16, 4, 2, news, [100, 40, 50], use_cu=news != [1, 1, 1], edit=edit)


def test_context_past_the_table_is_cut(P):
    gen = torch.Generator().manual_seed(1)
    kv = [x.cuda() for x in random_cache(gen, 4, 1, 16, 64)]
    q = torch.randn((1, 2, 64), generator=gen).half().cuda()
    t = i32([[2, 0]]).cuda()
    a = P.attention(q, kv, t, i32([32]).cuda())
    b = P.attention(q, kv, t, i32([1 << 30]).cuda())
    assert torch.equal(a, b)


@pytest.mark.parametrize("scale", [0.3, -0.2, 1e-4])
def test_scale(P, scale):
    check_attention(P, 1, 64, 16, 4, 2, [1, 9], [70, 100], scale=scale)


def test_peaked_and_flat_weights(P):
    check_attention(P, 1, 128, 16, 4, 2, [1, 1, 20], [600, 1300, 700], qscale=12.0)
    check_attention(P, 2, 128, 16, 4, 2, [1, 1, 20], [600, 1300, 700], qscale=0.01)


def test_shared_prefix_pages(P):
    """Two sequences that read the same pages see the same keys."""
    gen = torch.Generator().manual_seed(2)
    kv = [x.cuda() for x in random_cache(gen, 6, 2, 16, 64)]
    q = torch.randn((1, 4, 64), generator=gen).half().cuda().repeat(2, 1, 1)
    t = i32([[3, 1, 5], [3, 1, 5]]).cuda()
    out = P.attention(q, kv, t, i32([45, 45]).cuda())
    assert torch.equal(out[0], out[1])


def test_a_query_that_is_not_finite_spoils_only_itself(P):
    gen = torch.Generator().manual_seed(2)
    kv = [x.cuda() for x in random_cache(gen, 12, 2, 16, 64)]
    t, cu = R.make_tables(gen, [6, 5], 6, 12).cuda(), R.offsets([40, 1]).cuda()
    q = torch.randn((41, 4, 64), generator=gen).half().cuda()
    a = P.attention(q, kv, t, i32([90, 70]).cuda(), cu_seqlens=cu)
    q2 = q.clone()
    q2[7, 1, 5] = math.nan
    q2[40, 3, 5] = math.inf
    b = P.attention(q2, kv, t, i32([90, 70]).cuda(), cu_seqlens=cu)
    a[7, 1] = b[7, 1] = 0
    a[40, 3] = b[40, 3] = 0
    assert torch.equal(a, b)


def test_offsets_beyond_32_bits(P):
    """Pages whose elements lie behind 2^32 in the pool (10 GB of keys)."""
    D, page, Hkv = 256, 128, 8
    pages = 40000
    k = torch.empty((pages, Hkv, page, D), dtype=torch.int8, device="cuda")
    v = torch.empty_like(k)
    ks = torch.full((pages, Hkv), math.nan, device="cuda")
    vs = ks.clone()
    ids = [39999, 16400, 3, 33000]
    gen = torch.Generator().manual_seed(2)
    small = random_cache(gen, 4, Hkv, page, D)
    for i, p in enumerate(ids):
        k[p], v[p], ks[p], vs[p] = (x[i].cuda() for x in small)
    q = torch.randn((3, 8, D), generator=gen).half()
    t = i32([ids])
    out = P.attention(q.cuda(), (k, v, ks, vs), t.cuda(), i32([500]).cuda(), cu_seqlens=i32([0, 3]).cuda())
    near = P.attention(q.cuda(), gpu(*small), i32([[0, 1, 2, 3]]).cuda(), i32([500]).cuda(), cu_seqlens=i32([0, 3]).cuda())
    assert torch.equal(out, near)
    one = P.attention(q[:1].cuda(), (k, v, ks, vs), t.cuda(), i32([500]).cuda())
    near = P.attention(q[:1].cuda(), gpu(*small), i32([[0, 1, 2, 3]]).cuda(), i32([500]).cuda())
    assert torch.equal(one, near)
    rows = torch.randn((20, 8, D), generator=gen).half().cuda()
    near = gpu(*small)
    for kv, tab in (((k, v, ks, vs), t), (near, i32([[0, 1, 2, 3]]))):
        P.kv_append(rows, rows, kv, tab.cuda(), i32([490]).cuda(), 1e4, cu_seqlens=i32([0, 20]).cuda())
    for i, p in enumerate(ids):
        assert torch.equal(k[p], near[0][i]) and torch.equal(v[p], near[1][i]) and torch.equal(ks[p], near[2][i])
    a = P.kv_read((k, v, ks, vs), t.cuda(), i32([380]).cuda(), i32([0, 130]).cuda(), 130)
    b = P.kv_read(near, i32([[0, 1, 2, 3]]).cuda(), i32([380]).cuda(), i32([0, 130]).cuda(), 130)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


# --------------------------------------------------------------------------------------------------- ragged attention

def check_ragged(P, seed, D, Hq, Hkv, lengths, window=0, sink=0, scale=0.0, spoil=None, fused=True):
    gen = torch.Generator().manual_seed(seed)
    T = sum(lengths)
    rows = torch.randn((T, (Hq + 2 * Hkv) * D), generator=gen).half()
    if spoil:
        spoil(rows.view(T, Hq + 2 * Hkv, D))
    cut = lambda x: [x[:, a * D:b * D].unflatten(1, (b - a, D))  # noqa: E731
                     for a, b in ((0, Hq), (Hq, Hq + Hkv), (Hq + Hkv, Hq + 2 * Hkv))]
    q, k, v = cut(rows)
    dev = cut(rows.cuda())
    if not fused:
        dev = [x.contiguous() for x in dev]
    cu = R.offsets(lengths)
    out = P.attention_ragged(*dev, cu.cuda(), scale=scale, window=window, sink=sink)
    torch.cuda.synchronize()
    for b, n in enumerate(lengths):
        r = slice(int(cu[b]), int(cu[b]) + n)
        want, tol = R.attend(q[r], k[r], v[r], torch.arange(n), window, sink, scale)
        got = out[r].cpu().double()
        bad = ~torch.isfinite(want)
        assert bool((torch.isnan(got) == torch.isnan(want)).all()) and bool((got[bad & ~torch.isnan(want)] == want[bad & ~torch.isnan(want)]).all())
        err = (got - want).abs()
        assert bool((err <= tol)[~bad].all()), (b, n, float((err / tol)[~bad].max()))


RAGGED = [(64, 4, 2), (128, 2, 1), (256, 4, 1), (64, 9, 3), (128, 3, 3)]


@pytest.mark.parametrize("D,Hq,Hkv", RAGGED)
def test_ragged_lengths(P, D, Hq, Hkv):
    check_ragged(P, D + Hq, D, Hq, Hkv, [1, 2, 0, 15, 16, 17, 31, 33, 64, 65, 127, 130])


@pytest.mark.parametrize("D,Hq,Hkv", RAGGED)
@pytest.mark.parametrize("window,sink", [(1, 0), (31, 0), (64, 4), (100, 1), (20, 40), (500, 4), (129, 64)])
def test_ragged_window(P, D, Hq, Hkv, window, sink):
    check_ragged(P, window + D, D, Hq, Hkv, [70, 1, 210, 33], window, sink)


@pytest.mark.parametrize("D,Hq,Hkv,n", [(64, 2, 1, 700), (128, 2, 1, 513), (256, 1, 1, 600)])
@pytest.mark.parametrize("window,sink", [(0, 0), (130, 4)])
def test_ragged_long(P, D, Hq, Hkv, n, window, sink):
    check_ragged(P, n, D, Hq, Hkv, [n, 5], window, sink, fused=False)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("window,sink", [(0, 0), (40, 3)])
def test_what_is_not_seen_has_no_influence(P, D, window, sink):
    """NaN and infinities in keys and values: rows that see them show it as the formula says, all other rows - earlier
    ones, rows of other sequences, rows whose window has moved past them - are as if they were not there."""
    Hq, Hkv, lengths = 4, 2, [90, 37, 130]
    gen = torch.Generator().manual_seed(D)
    q, k, v = (torch.randn((sum(lengths), h, D), generator=gen).half().cuda() for h in (Hq, Hkv, Hkv))
    cu = R.offsets(lengths).cuda()
    clean = P.attention_ragged(q, k, v, cu, window=window, sink=sink)
    k2, v2 = k.clone(), v.clone()
    spots = [(50, 0), (100, 1), (127 + 20, 0), (127 + 64, 1)]       # row, kv head
    values = [math.nan, math.inf, -math.inf, math.nan]
    for (row, h), x in zip(spots, values):
        k2[row, h, 3] = x
        v2[row, h, 1] = x
        v2[row, h, D - 1] = -x
    out = P.attention_ragged(q, k2, v2, cu, window=window, sink=sink)
    touched = torch.zeros((sum(lengths), Hq), dtype=torch.bool)
    for row, h in spots:
        b = 0 if row < 90 else 1 if row < 127 else 2
        lo, n = [0, 90, 127][b], lengths[b]
        for i in range(n):
            if bool(R.seen(i, n, window, sink)[row - lo]):
                touched[lo + i, h * 2:h * 2 + 2] = True
    assert touched.any() and not touched.all()
    assert torch.equal(out.cpu()[~touched], clean.cpu()[~touched])


@pytest.mark.parametrize("D", [64, 128, 256])
def test_infinite_values_that_are_seen(P, D):
    """An infinity in a value row reaches every query that sees it, in its own column; two of different sign make NaN."""
    def spoil(rows):
        rows[3, 5, 7] = math.inf
        rows[20, 5, 7] = -math.inf
        rows[10, 4, 0] = math.nan
        rows[40, 5, 9] = math.inf
    # flat weights, so that none of them is zero in binary16
    check_ragged(P, 3, D, 4, 1, [70], scale=0.01, spoil=spoil)


def test_ragged_equals_paged_on_exact_codes(P):
    """Rows that INT8 codes with a power-of-two scale hold exactly: the two attentions compute the same thing."""
    gen = torch.Generator().manual_seed(2)
    n, D, Hq, Hkv, page = 75, 64, 4, 2, 16
    codes = lambda: torch.randint(-127, 128, (n, Hkv, D), generator=gen)  # noqa: E731
    kc, vc = codes(), codes()
    kc[::page, :, 0] = vc[::page, :, 0] = 127                     # every page reaches 127, its scale is 2^-6
    k, v = ((x.double() / 64).half().cuda() for x in (kc, vc))
    q = torch.randn((n, Hq, D), generator=gen).half().cuda()
    kv = P.empty_pages(6, Hkv, D, page)
    t, cu = i32([[4, 0, 2, 1, 5]]).cuda(), R.offsets([n]).cuda()
    P.kv_append(k, v, kv, t, i32([0]).cuda(), 0.0, cu_seqlens=cu)
    assert bool((kv[2][[4, 0, 2, 1, 5]] == 2.0 ** -6).all())
    for window, sink in ((0, 0), (20, 4)):
        a = P.attention(q, kv, t, i32([n]).cuda(), cu_seqlens=cu, window=window, sink=sink)
        b = P.attention_ragged(q, k, v, cu, window=window, sink=sink)
        _, tol = R.attend(q.cpu(), k.cpu(), v.cpu(), torch.arange(n), window, sink)
        assert bool(((a.double() - b.double()).cpu().abs() <= 2 * tol).all())


# --------------------------------------------------------------------------------------------------------- in a row

@pytest.mark.parametrize("D,Hq,Hkv,page,window,sink", [(64, 8, 2, 16, 0, 0), (128, 4, 2, 32, 60, 4)])
def test_prompt_then_tokens(P, D, Hq, Hkv, page, window, sink):
    """Prompts of three sequences (FP16 attention, rows into the cache), a second chunk of one of them, then tokens one by
    one: every step against the reference on the cache's own contents, and positions, pages and scales carried along."""
    gen = torch.Generator().manual_seed(page)
    B, theta, eps = 3, 1e4, 1e-6
    have = [0] * B
    width = 12
    kv = P.empty_pages(B * width, Hkv, D, page)
    tables = torch.randperm(B * width, generator=gen).int().reshape(B, width)
    td = tables.cuda()
    qw, kw = ((1 + 0.1 * torch.randn(D, generator=gen)).half() for _ in range(2))
    for news in ([50, 37, 0], [0, 40, 65], [1, 1, 1], [1, 1, 1], [1, 0, 1], [1, 1, 1]):
        T = sum(news)
        rows = torch.randn((T, (Hq + 2 * Hkv) * D), generator=gen).half()
        q, k, v = (rows.cuda()[:, a * D:b * D].unflatten(1, (b - a, D)) for a, b in
                   ((0, Hq), (Hq, Hq + Hkv), (Hq + Hkv, Hq + 2 * Hkv)))
        one = news == [1, 1, 1]
        cu = None if one else R.offsets(news).cuda()
        qr = P.kv_append(k, v, kv, td, i32(have).cuda(), theta, cu_seqlens=cu, q=q, q_weight=qw.cuda(), k_weight=kw.cuda(), eps=eps)
        total = [h + n for h, n in zip(have, news)]
        out = P.attention(qr, kv, td, i32(total).cuda(), cu_seqlens=cu, window=window, sink=sink)
        back = P.kv_read(kv, td, i32([0] * B).cuda(), R.offsets(total).cuda(), sum(total))
        at, rd = 0, 0
        for b in range(B):
            n, c = news[b], total[b]
            kk, _ = R.gather(kv[0].cpu(), kv[2].cpu(), tables[b], page, 0, c)
            vv, _ = R.gather(kv[1].cpu(), kv[3].cpu(), tables[b], page, 0, c)
            assert read_back(back[0][rd:rd + c], kk) and read_back(back[1][rd:rd + c], vv)
            want, tol = R.attend(qr[at:at + n].cpu(), kk, vv, torch.arange(have[b], c), window, sink, ratio=spread(kv[3].cpu()[tables[b].long()]))
            assert bool(((out[at:at + n].cpu().double() - want).abs() <= tol).all())
            # the newest rows are in the cache to within half a step of their page's scale
            x, terms = R.norm_rope(k[at:at + n].cpu(), kw, eps, theta, torch.arange(have[b], c))
            ids = tables[b, torch.arange(have[b], c) // page].long()
            assert bool(((kk[have[b]:] - x).abs() <= 0.5001 * kv[2].cpu().double()[ids][:, :, None] + terms * R.row_bound(D)).all())
            at, rd = at + n, rd + c
        have = total


def test_window_equals_the_ring_cache(P):
    """window = W - sink over pages against the contiguous cache's ring of W slots (kv_append_windowed +
    attention_hybrid_batched): both hold the same tokens, in codes of different scales."""
    import cactus_amd.hip as H
    gen = torch.Generator().manual_seed(5)
    D, Hq, Hkv, page, W, sink, steps = 128, 4, 2, 16, 40, 4, 70
    kc = torch.zeros((1, W, Hkv, D), dtype=torch.int8, device="cuda")
    vc, ks, vs = kc.clone(), torch.ones((1, W, Hkv, 1), device="cuda"), torch.ones((1, W, Hkv, 1), device="cuda")
    kv = P.empty_pages(5, Hkv, D, page)
    t = torch.randperm(5, generator=gen).int().reshape(1, 5).cuda()
    lens, pos = i32([0]).cuda(), i32([0]).cuda()
    for i in range(steps):
        q, k, v = (torch.randn((1, 1, h, D), generator=gen).half().cuda() for h in (Hq, Hkv, Hkv))
        ring = H.attention_hybrid_batched(q, kc, vc, ks, vs, k, v, 0.0, lens, pos)
        H.kv_append_windowed(k, v, kc, vc, ks, vs, pos, W, sink)
        P.kv_append(k[0], v[0], kv, t, i32([i]).cuda(), 0.0)
        paged = P.attention(q[0], kv, t, i32([i + 1]).cuda(), window=W - sink, sink=sink)
        H.kv_positions_advance(pos, lens, 1, W)
        # codes are off by half a step (|x| <= 5: 5 / 254 of it per element in either cache), weights follow the scores
        assert float((ring[0].float() - paged.float()).abs().max()) < 0.08


@pytest.mark.parametrize("shape", ["decode", "long", "chunk", "ragged"])
def test_captured_and_replayed(P, shape):
    """Replays with new inputs, eager work between them; every replay equals the eager call on the same inputs."""
    gen = torch.Generator().manual_seed(6)
    D, Hq, Hkv, page, width = 128, 4, 2, 16, 130
    news = {"decode": [1, 1, 1], "long": [1], "chunk": [40, 3, 70], "ragged": [40, 3, 70]}[shape]
    B, T = len(news), sum(news)
    past = {"decode": [40, 15, 100], "long": [2000], "chunk": [17, 0, 33], "ragged": [0, 0, 0]}[shape]
    kv = [x.cuda() for x in random_cache(gen, B * width, Hkv, page, D)]
    t = torch.randperm(B * width, generator=gen).int().reshape(B, width).cuda()
    cu = None if shape in ("decode", "long") else R.offsets(news).cuda()
    pos, ctx = i32(past).cuda(), i32([p + n for p, n in zip(past, news)]).cuda()
    x = [torch.zeros((T, h, D), dtype=torch.float16, device="cuda") for h in (Hq, Hkv, Hkv)]

    def step():
        q = P.kv_append(x[1], x[2], kv, t, pos, 1e4, cu_seqlens=cu, q=x[0])
        if shape == "ragged":
            return q, P.attention_ragged(q, x[1], x[2], cu)
        return q, P.attention(q, kv, t, ctx, cu_seqlens=cu)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q, out = step()
    for i in range(4):
        for y in x:
            y.copy_(torch.randn(y.shape, generator=gen).half())
        saved = [y.clone() for y in kv]
        graph.replay()
        torch.cuda.synchronize()
        got = [q.clone(), out.clone()] + [y.clone() for y in kv]
        for y, z in zip(kv, saved):
            y.copy_(z)
        want = list(step()) + [y.clone() for y in kv]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), i


def test_two_streams_at_once(P):
    """Calls on two streams that overlap do not meet: scratch belongs to the call."""
    gen = torch.Generator().manual_seed(7)
    D, Hq, Hkv, page = 128, 8, 2, 16
    kv = [x.cuda() for x in random_cache(gen, 600, Hkv, page, D)]
    jobs = []
    for i in range(2):
        t = torch.randperm(600, generator=gen)[:300].int().reshape(1, 300).cuda()
        q = torch.randn((1, Hq, D), generator=gen).half().cuda()
        jobs.append((q, kv, t, i32([4700 - 1000 * i]).cuda()))
    want = [P.attention(*j) for j in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(P.attention(*jobs[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])


def test_same_inputs_same_bits(P):
    gen = torch.Generator().manual_seed(8)
    D, Hq, Hkv, page = 64, 8, 2, 32
    kv = [x.cuda() for x in random_cache(gen, 200, Hkv, page, D)]
    t = R.make_tables(gen, [100, 60], 100, 200).cuda()
    q = torch.randn((60, Hq, D), generator=gen).half().cuda()
    runs = [P.attention(q, kv, t, i32([3100, 1900]).cuda(), cu_seqlens=R.offsets([59, 1]).cuda()) for _ in range(5)]
    ones = [P.attention(q[:2], kv, t, i32([3100, 1900]).cuda()) for _ in range(5)]
    assert all(torch.equal(runs[0], r) for r in runs) and all(torch.equal(ones[0], r) for r in ones)


def test_python_refuses(P):
    kv = P.empty_pages(4, 2, 64, 16)
    z = torch.zeros((1, 2, 64), dtype=torch.float16, device="cuda")
    t, one = i32([[0]]).cuda(), i32([1]).cuda()
    with pytest.raises(ValueError, match="q must be float16"):
        P.attention(z.float(), kv, t, one)
    with pytest.raises(ValueError, match="context_lens must be"):
        P.attention(z, kv, t, one.long())
    with pytest.raises(ValueError, match="heads of a row"):
        P.attention(z.transpose(1, 2).contiguous().transpose(1, 2), kv, t, one)
    with pytest.raises(ValueError, match="k must be float16"):
        P.kv_append(z[:, :1], z, kv, t, one, 1e4)
    with pytest.raises(ValueError, match="scales must be"):
        P.attention(z, (kv[0], kv[1], kv[2].half(), kv[3]), t, one)
    with pytest.raises(ValueError, match="must not be negative"):
        P.attention(z, kv, t, one, window=-1)
    with pytest.raises(Exception, match="multiple of the kv heads"):
        P.attention(torch.zeros((1, 3, 64), dtype=torch.float16, device="cuda"), kv, t, one)
    with pytest.raises(Exception, match="one row per sequence"):
        P.attention(torch.zeros((2, 2, 64), dtype=torch.float16, device="cuda"), kv, t, one)


# ------------------------------------------------------------------------------------------- what a caller may hand over

@pytest.mark.parametrize("news", [[1, 1, 1, 1], [40, 1, 70, 3]])
def test_lengths_that_are_not_lengths(P, news):
    """Context lengths are device data: below zero they are zero, above the table they end with it."""
    gen = torch.Generator().manual_seed(9)
    D, Hq, Hkv, page = 64, 4, 2, 16
    kv = [x.cuda() for x in random_cache(gen, 40, Hkv, page, D)]
    t = torch.randperm(40, generator=gen).int().reshape(4, 10).cuda()
    q = torch.randn((sum(news), Hq, D), generator=gen).half().cuda()
    cu = R.offsets(news).cuda() if news != [1, 1, 1, 1] else None
    for window, sink in ((0, 0), (30, 4), ((1 << 31) - 1, (1 << 31) - 1)):
        a = P.attention(q, kv, t, i32([-(1 << 31), -7, (1 << 31) - 1, 90]).cuda(), cu_seqlens=cu, window=window, sink=sink)
        b = P.attention(q, kv, t, i32([0, 0, 160, 90]).cuda(), cu_seqlens=cu, window=window, sink=sink)
        assert torch.equal(a, b)
        assert not a[:news[0] + news[1]].any()
        if window > 30:
            assert torch.equal(a, P.attention(q, kv, t, i32([0, 0, 160, 90]).cuda(), cu_seqlens=cu))


def test_sequence_offsets_that_are_not_offsets(P):
    """cu_seqlens is device data: whatever it holds, reads and writes stay inside the rows, and the calls end."""
    gen = torch.Generator().manual_seed(10)
    D, Hq, Hkv, page, T = 64, 4, 2, 16, 200
    kv = [x.cuda() for x in random_cache(gen, 60, Hkv, page, D)]
    t = torch.randperm(60, generator=gen).int().reshape(4, 15).cuda()
    rows = lambda h: torch.randn((T, h, D), generator=gen).half().cuda()  # noqa: E731
    q, k, v = rows(Hq), rows(Hkv), rows(Hkv)
    guard = torch.full((T + 400, Hq, D), 3.0, dtype=torch.float16, device="cuda")
    out = guard[200:200 + T]
    for bad in ([0, 90, 40, 150, 60], [50, 1 << 30, -5, (1 << 31) - 1, -(1 << 31)], [200, 150, 100, 50, 0], [-9, -8, -7, -6, -5]):
        cu = i32(bad).cuda()
        P.attention_ragged(q, k, v, cu, out=out)
        P.attention(q, kv, t, i32([100, 240, 3, 77]).cuda(), cu_seqlens=cu, out=out)
        P.kv_append(k, v, kv, t, i32([0, 20, 5, 1000]).cuda(), 1e4, cu_seqlens=cu, q=q, out_q=out)
        k2, v2 = guard[:0].new_full((T + 2, Hkv, D), 3.0), guard[:0].new_full((T + 2, Hkv, D), 3.0)
        P.kv_read(kv, t, i32([0, 20, -5, 1000]).cuda(), cu, T, out_k=k2[1:-1], out_v=v2[1:-1])
        torch.cuda.synchronize()
        assert bool((guard[:200] == 3.0).all()) and bool((guard[200 + T:] == 3.0).all())
        assert all(bool((x[0] == 3.0).all()) and bool((x[-1] == 3.0).all()) for x in (k2, v2))


@pytest.mark.parametrize("D,news,contexts", [(64, [1, 1], [300, 47]), (128, [1, 1], [300, 47]), (256, [1, 1], [300, 47]),
                                             (64, [70, 40], [300, 120]), (128, [70, 40], [300, 120]), (256, [30, 40], [200, 120])])
def test_page_scales_far_apart(P, D, news, contexts):
    """Scales from zero over the smallest that append makes to large ones, side by side.  A weight is rounded to binary16 together
    with its page's value scale, beside the largest such product: where it is subnormal it is off by 2^-25 of that, times a
    code of at most 127, for each key."""
    gen = torch.Generator().manual_seed(11)
    Hq, Hkv, page = 4, 2, 16
    used = [(c + page - 1) // page for c in contexts]
    total = sum(used)
    kv = list(random_cache(gen, total, Hkv, page, D))
    pick = lambda xs: torch.tensor(xs)[torch.randint(0, len(xs), (total, Hkv), generator=gen)]  # noqa: E731
    kv[2], kv[3] = pick([0.0, 1e-10, 1e-3, 0.02, 0.05]), pick([0.0, 1e-10, 1e-4, 0.02, 2.0])
    t = R.make_tables(gen, used, max(used), total)
    q = torch.randn((sum(news), Hq, D), generator=gen).half()
    cu = R.offsets(news)
    out = P.attention(q.cuda(), [x.cuda() for x in kv], t.cuda(), i32(contexts).cuda(), cu_seqlens=cu.cuda()).cpu().double()
    for b, (n, c) in enumerate(zip(news, contexts)):
        k, ok = R.gather(kv[0], kv[2], t[b], page, 0, c)
        v, _ = R.gather(kv[1], kv[3], t[b], page, 0, c)
        r = slice(int(cu[b]), int(cu[b]) + n)
        want, tol = R.attend(q[r], k, v, torch.arange(c - n, c), 0, 0, 0.0, ok)
        tol = tol + 2.0 ** -25 * 2.0 * 127 * c
        assert bool(((out[r] - want).abs() <= tol).all()), (b, float(((out[r] - want).abs() / tol).max()))


@pytest.mark.parametrize("D,Hq,Hkv,n", [(64, 8, 2, 1100), (128, 8, 4, 1100), (256, 4, 1, 1100), (64, 12, 3, 2100)])
@pytest.mark.parametrize("window,sink", [(0, 0), (200, 4)])
def test_ragged_many_tiles(P, D, Hq, Hkv, n, window, sink):
    """More row tiles than the order of the workgroups deals out at a time, whatever the number of kv heads; some rows of each
    sequence are checked."""
    gen = torch.Generator().manual_seed(n + D)
    lengths = [3, n, 0, n // 3]
    T = sum(lengths)
    q, k, v = (torch.randn((T, h, D), generator=gen).half() for h in (Hq, Hkv, Hkv))
    cu = R.offsets(lengths)
    out = P.attention_ragged(q.cuda(), k.cuda(), v.cuda(), cu.cuda(), window=window, sink=sink).cpu().double()
    assert bool(torch.isfinite(out).all())
    for b, m in enumerate(lengths):
        rows = torch.arange(m) if m < 8 else torch.cat([torch.arange(0, m, 61), torch.tensor([m - 1])])
        base = int(cu[b])
        want, tol = R.attend(q[base + rows], k[base:base + m], v[base:base + m], rows, window, sink)
        assert bool(((out[base + rows] - want).abs() <= tol).all()), b


@pytest.mark.parametrize("D,page,Hq,Hkv", [(64, 16, 4, 2), (128, 64, 4, 2), (256, 128, 2, 1)])
@pytest.mark.parametrize("window,sink", [(0, 0), (1500, 4), (2000, 100)])
def test_chunk_over_a_long_context(P, D, page, Hq, Hkv, window, sink):
    check_attention(P, D, D, page, Hq, Hkv, [50, 33], [3100, 1700], window, sink)


def test_row_strides_of_a_wide_matrix(P):
    """Rows that are columns of a matrix as wide as a stride may be: offsets inside a tile pass 2^30 bytes."""
    gen = torch.Generator().manual_seed(12)
    D, n, stride = 64, 130, (1 << 24) - 8
    pool = torch.zeros(n * stride // 2, dtype=torch.float32, device="cuda").view(torch.float16)
    at = [pool.as_strided((n, h, D), (stride, D, 1), o) for h, o in ((2, 0), (1, 1024), (1, 4096))]
    x = [torch.randn((n, h, D), generator=gen).half().cuda() for h in (2, 1, 1)]
    for a, b in zip(at, x):
        a.copy_(b)
    cu = i32([0, n]).cuda()
    assert torch.equal(P.attention_ragged(*at, cu), P.attention_ragged(*x, cu))


def test_two_graphs_replayed_side_by_side(P):
    """Two captured calls with scratch of their own, replayed on two streams at once and in turn."""
    gen = torch.Generator().manual_seed(13)
    D, Hq, Hkv, page, width = 128, 4, 2, 16, 250
    kv = [x.cuda() for x in random_cache(gen, 2 * width, Hkv, page, D)]
    t = torch.randperm(2 * width, generator=gen).int().reshape(2, 1, width).cuda()
    q = [torch.randn((1, Hq, D), generator=gen).half().cuda() for _ in range(2)]
    ctx = [i32([3900]).cuda(), i32([2500]).cuda()]
    graphs, outs = [], []
    for i in range(2):
        P.attention(q[i], kv, t[i], ctx[i])
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(P.attention(q[i], kv, t[i], ctx[i]))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for turn in range(5):
        for x in q:
            x.copy_(torch.randn(x.shape, generator=gen).half())
        torch.cuda.synchronize()
        if turn < 3:
            for g, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
        else:
            for g in graphs[::-1]:
                g.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in outs]
        want = [P.attention(q[i], kv, t[i], ctx[i]) for i in range(2)]
        assert all(torch.equal(a, b) for a, b in zip(got, want)), turn


@pytest.mark.parametrize("batch", [2, 17, 63, 64, 65, 130])
@pytest.mark.parametrize("D,Hq,Hkv,longest", [(64, 4, 2, 150), (128, 2, 1, 200), (256, 8, 1, 20)])
def test_batches_of_every_size(P, batch, D, Hq, Hkv, longest):
    """Chunks beside single tokens and sequences that bring nothing; long and short contexts (split keys), prompts too."""
    gen = torch.Generator().manual_seed(batch + D)
    news = [int(x) for x in torch.randint(0, 4, (batch,), generator=gen)]
    for b, n in ((batch // 3, longest), (batch - 1, longest // 2 + 1), (0, 17)):
        news[b] = n
    contexts = [n + int(x) for n, x in zip(news, torch.randint(0, 40, (batch,), generator=gen))]
    contexts[batch // 3] += 1100
    contexts[batch - 1] += 600
    check_attention(P, batch, D, 32, Hq, Hkv, news, contexts)
    check_ragged(P, batch, D, Hq, Hkv, news, 40, 3)


@pytest.mark.parametrize("batch", [1000, 1024, 1025])
def test_batches_of_a_thousand(P, batch):
    gen = torch.Generator().manual_seed(batch)
    news = [int(x) for x in torch.randint(0, 2, (batch,), generator=gen)]
    news[0], news[500], news[batch - 1] = 20, 70, 33
    contexts = [n + int(x) for n, x in zip(news, torch.randint(0, 20, (batch,), generator=gen))]
    contexts[500] += 1100
    check_attention(P, batch, 64, 16, 2, 1, news, contexts)
    check_ragged(P, batch, 64, 2, 1, news)


@pytest.mark.parametrize("Hq,Hkv", [(16, 1), (40, 2), (64, 1), (130, 1), (14, 7)])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_chunks_of_wide_groups(P, D, Hq, Hkv):
    """More query heads per kv head than a wave or a tile has rows."""
    check_attention(P, Hq + D, D, 16, Hq, Hkv, [5, 1, 3], [40, 70, 3], 30, 2)
    check_ragged(P, Hq + D, D, Hq, Hkv, [7, 1, 20], 6, 1)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("window,sink", [(0, 0), (100, 4)])
def test_ragged_launches_that_fill_the_chip(P, D, window, sink):
    """Enough row tiles x kv heads that one group of waves takes all keys of a tile; a value that is not finite spoils the rows that
    see it, in its dim, and no others."""
    gen = torch.Generator().manual_seed(D + window)
    H, lengths = 40, [300, 1400]
    T = sum(lengths)
    q, k, v = (torch.randn((T, H, D), generator=gen).half() for _ in range(3))
    v[300 + 650, :, 5], v[300 + 651, :, 6], k[300 + 1390] = math.nan, math.inf, math.nan
    cu = R.offsets(lengths)
    out = P.attention_ragged(q.cuda(), k.cuda(), v.cuda(), cu.cuda(), window=window, sink=sink).cpu().double()
    for b, m in enumerate(lengths):
        rows = torch.tensor(sorted({0, 1, m - 1, *range(7, m, 61), *(x for x in (649, 650, 651, 700, 750, 751, 752, 1389) if x < m)}))
        rows = rows[rows < 1390]
        base = int(cu[b])
        want, tol = R.attend(q[base + rows], k[base:base + m], v[base:base + m], rows, window, sink)
        got, fine = out[base + rows], torch.isfinite(want)
        assert bool((torch.isfinite(got) == fine).all()), b
        assert bool((got[~fine & ~torch.isnan(want)] == want[~fine & ~torch.isnan(want)]).all())
        assert bool(((got - want).abs() <= tol)[fine].all()), b
