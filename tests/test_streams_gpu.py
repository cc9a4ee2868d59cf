"""GPU: the operators that serve streams of different lengths from one paged cache (include/avt_hip.h, ABI 10), each against a plain evaluation in 64 bits
(whole numbers: in Python), and a run of them together through AVTh's streams.

Tolerances.  u = eps(bf16) / 2 = 2^-8 is the half step of the output's rounding and of the probabilities' before the second product:
  attention   |o - ref| <= u |ref| + (u + 2 ds + 2^-16) A,  A = sum_j p_j |v_j| (what an error of p's size can move) + the same u for the sum the rounding
              of the output meets; ds = hd 2^-24 scale max_j sum_d |q_d k_jd| bounds the error of a score summed in fp32 (hd additions of half steps), it enters p
              and the sum (2 ds); 2^-16 covers exp (arguments to 2^6, each off by a half step 2^-24, its own error 2^-21) and the fp32 sums of up to 2^8 partial results.
  w4          |y - ref| <= u |ref| + K 2^-23 B,  B = sum |x| s |u - 8| + the offset's part 24 sum |x| s (K additions of half steps 2^-24, twice for offset and groups);
              the tanh GELU's slope is at most 1.13 and its own error below 2^-18 of its argument."""
import math
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))

from avt_amd.lib import AvtHipError

pytestmark = pytest.mark.gpu
U = 2.0 ** -8
BF16, I32 = torch.bfloat16, torch.int32


@pytest.fixture(scope='module')
def ops():
    from avt_amd import ops as o
    return o


def i32(x):
    return torch.tensor(x, device='cuda', dtype=I32)


# ---- plan --------------------------------------------------------------------------------------------------------------------------------------
def plan_in_python(lens, new, owned, table, free, n_free, page, tokens):
    R, width = len(lens), len(table[0])
    table = [list(r) for r in table]
    n_free = max(0, min(n_free, len(free)))
    cu, kv, own, slots, pos, st, need_sum, taken = [0], [], [], [-1] * tokens, [-1] * tokens, [-1] * tokens, 0, 0
    for r in range(R):
        n = max(new[r], 0)
        start, end = cu[-1], sum(max(v, 0) for v in new[:r + 1])
        pages = -(-(lens[r] + n) // page)
        fits = pages <= width and end <= tokens
        need = max(0, pages - owned[r]) if fits else 0
        ok = fits and (need == 0 or need_sum + need <= n_free)
        if ok:
            for j in range(need):
                table[r][owned[r] + j] = free[n_free - 1 - need_sum - j]
            taken += need
        need_sum += need
        kv.append(lens[r] + n if ok else 0)
        own.append(owned[r] + (need if ok else 0))
        for i in range(n):
            if start + i < tokens:
                p = lens[r] + i
                st[start + i], pos[start + i] = r, p
                if ok:
                    slots[start + i] = table[r][p // page] * page + p % page
        cu.append(min(end, tokens))
    return cu, kv, own, [n_free - taken], slots, pos, st, table


def make_plan(R, new_max, past_max, page, seed, spare=5, extra_rows=0, width_less=0):
    g = torch.Generator().manual_seed(seed)
    new = torch.randint(0, new_max + 1, (R,), generator=g).tolist()
    lens = torch.randint(0, past_max + 1, (R,), generator=g).tolist()
    owned = [-(-l // page) + (1 if i % 3 == 0 else 0) for i, l in enumerate(lens)]
    width = max(1, max(max(o, -(-(l + n) // page)) for o, l, n in zip(owned, lens, new)) - width_less)
    owned = [min(o, width) for o in owned]
    lens = [min(l, o * page) for l, o in zip(lens, owned)]
    need = sum(max(0, -(-(l + n) // page) - o) for l, n, o in zip(lens, new, owned))
    perm = torch.randperm(sum(owned) + max(need + spare, 0), generator=g).tolist()
    table, at = [], 0
    for o in owned:
        table.append(perm[at:at + o] + [-7] * (width - o))
        at += o
    free = perm[at:]
    return lens, new, owned, table, free, len(free), page, sum(new) + extra_rows


@pytest.mark.parametrize('R,new_max,past_max,page,spare,extra,less', [
    (1, 1, 0, 8, 3, 0, 0), (1, 700, 50, 16, 0, 3, 0), (3, 1, 14, 16, 0, 0, 0), (3, 0, 14, 16, 0, 2, 0), (64, 9, 300, 64, 1, 0, 0), (65, 33, 300, 1024, 0, 5, 0),
    (1023, 5, 90, 16, 2, 0, 0), (1025, 3, 200, 32, 0, 1, 0), (4096, 2, 40, 8, 0, 0, 0), (37, 400, 100, 128, 0, 0, 0),
    (50, 20, 100, 16, -6, 0, 0), (50, 20, 100, 16, -400, 0, 0), (50, 20, 100, 16, 5, 0, 3), (50, 20, 100, 16, 5, -40, 0), (300, 40, 100, 16, -100, -900, 2)])
def test_plan_equals_the_plain_loop(ops, R, new_max, past_max, page, spare, extra, less):
    """Whole numbers: equal.  With streams that take nothing, more tokens than fit, too few pages (spare < 0), a table too narrow for some, rows too few for some."""
    a = make_plan(R, new_max, past_max, page, 7 * R + page, spare, extra, less)
    lens, new, owned, table, free, n_free, page, tokens = a
    want = plan_in_python(*a)
    dev = [i32(lens), i32(new), i32(owned), i32(table), i32(free), i32([n_free])]
    before = [d.clone() for d in dev]
    for _ in range(2):                                  # the same call again finds the same (the table's new entries are written again)
        p = ops.paged_plan(*dev, page, tokens)
        got = [p.cu, p.kv_lens, p.owned, p.n_free, p.slots, p.positions, p.streams, dev[3]]
        for name, x, y in zip('cu kv_lens owned n_free slots positions streams table'.split(), got, want):
            assert x.tolist() == y, name
    for i in (0, 1, 2, 4, 5):
        assert torch.equal(dev[i], before[i])


def test_plan_takes_a_wider_table_and_clamps_the_stack(ops):
    a = make_plan(20, 9, 100, 16, 3)
    lens, new, owned, table, free, n_free, page, tokens = a
    big = torch.full((20, len(table[0]) + 9), -3, device='cuda', dtype=I32)
    big[:, :len(table[0])] = i32(table)
    view = big[:, :len(table[0])]
    p = ops.paged_plan(i32(lens), i32(new), i32(owned), view, i32(free), i32([10 ** 6]), page, tokens)      # more than the stack holds: what it holds
    want = plan_in_python(*a)
    assert p.slots.tolist() == want[4] and view.tolist() == want[7] and p.n_free.tolist() == want[3]
    assert bool((big[:, len(table[0]):] == -3).all())


def test_plan_refuses(ops):
    ok = [i32([3]), i32([1]), i32([1]), i32([[0, 0]]), i32([5]), i32([1])]
    ops.paged_plan(*ok, 16, 1)
    for i, bad in ((0, i32([3]).long()), (1, i32([1, 2])), (2, i32([1]).float()), (3, i32([0, 0])), (3, i32([[0], [0]])), (5, i32([1, 1])), (4, i32([5]).cpu())):
        args = list(ok)
        args[i] = bad
        with pytest.raises(AvtHipError):
            ops.paged_plan(*args, 16, 1)
    for page in (0, 4, 24, 2048, -16):
        with pytest.raises(AvtHipError, match='page'):
            ops.paged_plan(*ok, page, 1)
    with pytest.raises(AvtHipError, match='streams'):
        ops.paged_plan(i32([0] * 5000), i32([1] * 5000), i32([0] * 5000), i32([[0]] * 5000), i32([0]), i32([1]), 16, 5000)
    with pytest.raises(AvtHipError):
        ops.paged_plan(*ok, 16, -1)


# ---- write -------------------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize('T,H,hd,page,fused', [(1, 4, 512, 16, True), (3, 1, 8, 8, False), (64, 4, 512, 16, True), (1000, 8, 64, 32, True), (257, 3, 40, 128, False), (4099, 2, 128, 64, True)])
def test_write_puts_rows_into_their_slots(ops, T, H, hd, page, fused):
    g = torch.Generator(device='cuda').manual_seed(T)
    P = T // page + 3
    kc, vc = (torch.randn((P, page, H, hd), generator=g, device='cuda').to(BF16) for _ in range(2))
    if fused:
        qkv = torch.randn((T, 3 * H * hd), generator=g, device='cuda').to(BF16)
        k, v = qkv[:, H * hd:2 * H * hd].view(T, H, hd), qkv[:, 2 * H * hd:].view(T, H, hd)
    else:
        k, v = (torch.randn((T, H, hd), generator=g, device='cuda').to(BF16) for _ in range(2))
    slots = torch.randperm(P * page, generator=g, device='cuda')[:T].to(I32)
    slots[T // 2] = -1
    if T > 2:
        slots[0], slots[T - 1] = P * page, -2 ** 31          # outside the cache: nothing is written
    wk, wv = kc.clone(), vc.clone()
    at = slots.tolist()
    for t, s in enumerate(at):
        if 0 <= s < P * page:
            wk.view(-1, H, hd)[s], wv.view(-1, H, hd)[s] = k[t], v[t]
    ops.paged_kv_write(k, v, kc, vc, slots)
    assert torch.equal(kc.view(torch.int16), wk.view(torch.int16)) and torch.equal(vc.view(torch.int16), wv.view(torch.int16))


def test_write_refuses_and_takes_nothing(ops):
    kc, vc = (torch.zeros((2, 16, 2, 64), device='cuda', dtype=BF16) for _ in range(2))
    k = torch.ones((3, 2, 64), device='cuda', dtype=BF16)
    s = i32([0, 1, 2])
    ops.paged_kv_write(k[:0], k[:0], kc, vc, s[:0])
    assert not kc.any()
    for args in ((k.float(), k, kc, vc, s), (k, k, kc, vc[:1], s), (k, k, kc.transpose(0, 1), vc.transpose(0, 1), s), (k, k, kc, vc, s[:2]), (k, k, kc, vc, s.long()),
                 (k[:, :1], k[:, :1], kc, vc, s), (k.transpose(0, 1).contiguous().transpose(0, 1), k, kc, vc, s), (k, k, kc, vc, s.cpu()), (k.cpu(), k.cpu(), kc.cpu(), vc.cpu(), s.cpu())):
        with pytest.raises(AvtHipError):
            ops.paged_kv_write(*args)
    odd = torch.ones((3, 3 * 2 * 64 + 4), device='cuda', dtype=BF16)[:, 4:132].view(3, 2, 64)                                  # rows that do not begin on 16 bytes
    with pytest.raises(AvtHipError, match='16-byte'):
        ops.paged_kv_write(odd, odd, kc, vc, s)


# ---- attention ---------------------------------------------------------------------------------------------------------------------------------
def attn_in_64(q, kc, vc, table, cu, kv_lens, scale):
    """(ref, bound) on the device in 64 bits: bound = the tolerance of the header comment."""
    T, H, hd = q.shape
    P, page, Hkv, _ = kc.shape
    grp = H // Hkv
    ref = torch.zeros((T, H, hd), device='cuda', dtype=torch.float64)
    tol = torch.full((T, H, hd), 1e-30, device='cuda', dtype=torch.float64)
    width = table.size(1)
    for r in range(len(kv_lens)):
        n, kv = cu[r + 1] - cu[r], min(kv_lens[r], width * page)
        if n == 0 or kv == 0:
            continue
        tok = torch.arange(kv, device='cuda')
        pg = table[r].long()[tok // page]
        there = (pg >= 0) & (pg < P)
        pg = pg.clamp(0, P - 1)
        x = kv - n + torch.arange(n, device='cuda')
        see = (tok[None] <= x[:, None]) & there[None]
        for h in range(H):
            K, V = kc[pg, tok % page, h // grp].double(), vc[pg, tok % page, h // grp].double()
            Q = q[cu[r]:cu[r] + n, h].double()
            s = (Q @ K.t().contiguous()) * scale
            s = torch.where(see, s, -math.inf)
            mag = torch.where(see, (Q.abs() @ K.abs().t().contiguous()) * scale, 0.0).nan_to_num(0.0).amax(1)
            m = s.amax(1, keepdim=True)
            p = torch.where(see, torch.exp(s - torch.where(m > -math.inf, m, 0.0)), 0.0)
            den = p.sum(1, keepdim=True)
            p = torch.where(den > 0, p / den, 0.0)
            vis = see.any(0)
            Vz = torch.where(vis[:, None], V, 0.0)
            o, A = p @ Vz, p @ Vz.abs()
            ref[cu[r]:cu[r] + n, h] = o
            ds = hd * 2.0 ** -24 * mag[:, None]
            tol[cu[r]:cu[r] + n, h] += U * o.abs() + (U + 2 * ds + 2.0 ** -16) * A
    return ref.view(T, H * hd), tol.view(T, H * hd)


def make_attn(new, kv, H, Hkv, hd, page, seed, spare_width=0, rows_behind=0, strided=True, junk=float('nan'), scale=1.0):
    """Caches whose rows behind each stream's tokens, and whose unused pages, hold `junk`."""
    g = torch.Generator(device='cuda').manual_seed(seed)
    have = [-(-k // page) for k in kv]
    P = sum(have) + 2
    perm = torch.randperm(P, generator=g, device='cuda').tolist()
    width = max(1, max(have) + spare_width)
    table, at = [], 0
    kc, vc = (torch.full((P, page, Hkv, hd), junk, device='cuda', dtype=BF16) for _ in range(2))
    for h, k in zip(have, kv):
        pages = perm[at:at + h]
        at += h
        for i, pg in enumerate(pages):
            n = min(page, k - i * page)
            kc[pg, :n] = (torch.randn((n, Hkv, hd), generator=g, device='cuda') * scale).to(BF16)
            vc[pg, :n] = torch.randn((n, Hkv, hd), generator=g, device='cuda').to(BF16)
        table.append(pages + [perm[-1]] * (width - h))
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    T = cu[-1] + rows_behind
    if strided:
        q = torch.randn((T, (H + 2 * Hkv) * hd), generator=g, device='cuda').to(BF16)[:, :H * hd].view(T, H, hd)
    else:
        q = torch.randn((T, H, hd), generator=g, device='cuda').to(BF16)
    return q, kc, vc, i32(table), cu, kv


def check_attn(ops, q, kc, vc, table, cu, kv, scale=None, **kw):
    hd = q.size(2)
    ref, tol = attn_in_64(q, kc, vc, table, cu, kv, hd ** -0.5 if scale is None else scale)
    out = torch.full((q.size(0), q.size(1) * hd), 7.0, device='cuda', dtype=BF16)
    got = ops.paged_attn(q, kc, vc, table, i32(cu), i32(kv), scale=scale, out=out, **kw)
    assert got is out
    T = cu[-1]
    over = ((out[:T].double() - ref[:T]).abs() - tol[:T])
    assert bool(torch.isfinite(out[:T]).all())
    assert float(over.max()) <= 0 if T else True, (float(over.max()), float((out[:T].double() - ref[:T]).abs().max()))
    assert bool((out[T:] == 7.0).all())              # rows behind the last stream are left as they were
    return out


HEADS = [(4, 4, 512), (2, 2, 1024), (12, 12, 64), (8, 2, 128), (8, 1, 256), (3, 3, 40), (16, 2, 64), (5, 5, 8), (32, 2, 128), (2, 1, 136), (4, 2, 520)]


@pytest.mark.parametrize('H,Hkv,hd', HEADS)
def test_attention_of_one_new_token(ops, H, Hkv, hd):
    kv = [1, 2, 15, 16, 17, 31, 33, 64, 65, 200, 513, 1000]
    a = make_attn([1] * len(kv), kv, H, Hkv, hd, 16, H * hd)
    check_attn(ops, *a)
    check_attn(ops, *a, max_new=1, max_kv=1000)


@pytest.mark.parametrize('H,Hkv,hd', HEADS)
def test_attention_of_chunks(ops, H, Hkv, hd):
    new = [1, 7, 40, 0, 3, 129, 64, 2]
    kv = [30, 7, 100, 50, 64, 300, 65, 700]
    a = make_attn(new, kv, H, Hkv, hd, 32, hd + H, spare_width=3, rows_behind=5)
    check_attn(ops, *a)
    check_attn(ops, *a, max_new=129, max_kv=700)


@pytest.mark.parametrize('H,Hkv,hd,page', [(4, 4, 512, 16), (8, 2, 128, 64), (8, 8, 64, 8), (4, 1, 256, 1024), (8, 2, 64, 128)])
def test_attention_of_long_chunks(ops, H, Hkv, hd, page):
    a = make_attn([515, 1, 258], [515, 1500, 1031], H, Hkv, hd, page, 3 * hd)
    check_attn(ops, *a)
    check_attn(ops, *a, max_new=515, max_kv=1500)


@pytest.mark.parametrize('hint', [(0, 0), (1, 1), (1, 3000), (3000, 1), (10 ** 9, 10 ** 9), (1, 10 ** 9)])
def test_hints_change_no_result(ops, hint):
    """max_new / max_kv choose kernels and grids only: also a caller that is wrong about them gets the attention."""
    a = make_attn([1, 90, 300, 2], [2500, 90, 1300, 40], 4, 2, 128, 16, 5)
    check_attn(ops, *a, max_new=hint[0], max_kv=hint[1])


@pytest.mark.parametrize('hd', [64, 128, 512])
def test_rows_that_see_nothing_are_zero(ops, hd):
    """A refused stream (kv_lens 0), fewer cached tokens than new ones, a stream without new tokens, one whose pages are not there."""
    q, kc, vc, table, cu, kv = make_attn([4, 20, 0, 3, 5], [30, 40, 10, 3, 60], 4, 4, hd, 16, 9)
    kv = [30, 0, 10, 2, 60]
    table[4, 1] = -1
    table[4, 3] = kc.size(0)
    out = check_attn(ops, q, kc, vc, table, cu, kv)
    assert not out[4:24].any() and not out[24].any()
    table[4] = -5
    out = check_attn(ops, q, kc, vc, table, cu, kv)
    assert not out[27:32].any()


@pytest.mark.parametrize('H,Hkv,hd', [(4, 4, 512), (8, 2, 128), (12, 12, 64), (4, 1, 256)])
@pytest.mark.parametrize('bad', [float('nan'), float('inf'), -float('inf')])
def test_what_a_row_does_not_see_has_no_influence(ops, H, Hkv, hd, bad):
    """The last cached token's key and value are not finite: every earlier row of its stream is as if they were not there."""
    new, kv = [70, 3, 200], [100, 64, 230]
    q, kc, vc, table, cu, kv = make_attn(new, kv, H, Hkv, hd, 16, 17)
    for r, k in enumerate(kv):
        pg = int(table[r, (k - 1) // 16])
        kc[pg, (k - 1) % 16] = bad
        vc[pg, (k - 1) % 16] = bad
    out = ops.paged_attn(q, kc, vc, table, i32(cu), i32(kv))
    ref, tol = attn_in_64(q, torch.nan_to_num(kc, 0, 0, 0), torch.nan_to_num(vc, 0, 0, 0), table, cu, kv, hd ** -0.5)
    for r in range(len(new)):
        lo, hi = cu[r], cu[r + 1] - 1
        assert bool(torch.isfinite(out[lo:hi]).all())
        assert float(((out[lo:hi].double() - ref[lo:hi]).abs() - tol[lo:hi]).max()) <= 0
        assert bad != bad and bool(torch.isnan(out[hi]).all()) or bad == bad      # (a NaN that IS seen is passed on)


def test_a_value_that_is_not_finite_reaches_exactly_its_column(ops):
    q, kc, vc, table, cu, kv = make_attn([70], [100], 4, 2, 128, 16, 23)
    pg = int(table[0, 50 // 16])
    vc[pg, 50 % 16, 1, 9] = float('inf')
    out = ops.paged_attn(q, kc, vc, table, i32(cu), i32(kv)).view(70, 4, 128)
    hit = torch.zeros((70, 4, 128), dtype=torch.bool, device='cuda')
    hit[20:, 2:, 9] = True                                     # rows at positions 50 and later, the heads of kv head 1, column 9
    assert torch.equal(torch.isinf(out), hit) and bool(torch.isfinite(out[~hit]).all())


@pytest.mark.parametrize('scale', [0.0, 1.0, -0.3])
def test_scales_and_large_scores(ops, scale):
    a = make_attn([33, 1], [200, 900], 4, 4, 64, 16, 31, scale=4.0)
    check_attn(ops, *a, scale=scale)


def test_equal_keys_average_and_runs_repeat(ops):
    q, kc, vc, table, cu, kv = make_attn([1, 60], [800, 500], 8, 2, 128, 16, 41)
    a = ops.paged_attn(q, kc, vc, table, i32(cu), i32(kv))
    for _ in range(3):
        assert torch.equal(a, ops.paged_attn(q, kc, vc, table, i32(cu), i32(kv)))      # no atomics: the same bits


def test_many_streams(ops):
    """More streams than a wave probes in two steps, most of them without new tokens."""
    R = 4200
    new = [1 if r % 5 == 0 else 0 for r in range(R)]
    kv = [1 + r % 40 for r in range(R)]
    check_attn(ops, *make_attn(new, kv, 2, 2, 64, 8, 51, junk=0.0))


def test_attention_on_another_stream_and_in_two_graphs(ops):
    """Two captured steps of different sizes, replayed in turns with eager work between; every replay equals the eager result."""
    runs = [make_attn([1] * 8, [100 * i + 90 for i in range(8)], 4, 2, 128, 16, 61), make_attn([40, 3], [640, 1100], 4, 2, 128, 16, 62)]
    want, graphs = [], []
    for q, kc, vc, table, cu, kv in runs:
        want.append(ops.paged_attn(q, kc, vc, table, i32(cu), i32(kv), max_kv=1100))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for (q, kc, vc, table, cu, kv), w in zip(runs, want):
            got = ops.paged_attn(q, kc, vc, table, i32(cu), i32(kv), max_kv=1100)
            side.synchronize()
            assert torch.equal(got, w)
    for q, kc, vc, table, cu, kv in runs:
        cud, kvd = i32(cu), i32(kv)
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = ops.paged_attn(q, kc, vc, table, cud, kvd, max_kv=1100)
        graphs.append((gr, out, cud, kvd))
    for _ in range(3):
        for (gr, out, _, _), w in zip(graphs, want):
            out.fill_(0)
            gr.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, w)
    gr, out, cud, kvd = graphs[0]
    kvd.sub_(3)                                               # the lengths live on the device: a replay takes the ones it finds
    gr.replay()
    torch.cuda.synchronize()
    q, kc, vc, table, cu, kv = runs[0]
    assert torch.equal(out, ops.paged_attn(q, kc, vc, table, i32(cu), i32([k - 3 for k in kv]), max_kv=1100))


def test_attention_refuses_and_takes_nothing(ops):
    q, kc, vc, table, cu, kv = make_attn([2, 3], [20, 30], 4, 2, 64, 16, 71)
    cud, kvd = i32(cu), i32(kv)
    assert ops.paged_attn(q[:0], kc, vc, table, i32([0, 0, 0]), kvd).shape == (0, 256)
    for args in ((q.float(), kc, vc, table, cud, kvd), (q, kc, vc[:1], table, cud, kvd), (q, kc.float(), vc.float(), table, cud, kvd), (q, kc, vc, table.long(), cud, kvd),
                 (q, kc, vc, table, cud[:2], kvd), (q, kc, vc, table[:1], cud, kvd), (q, kc, vc, table, cud.long(), kvd), (q[:, :3], kc, vc, table, cud, kvd),
                 (q[:, :, :32], kc, vc, table, cud, kvd), (q, kc.transpose(0, 1), vc.transpose(0, 1), table, cud, kvd), (q, kc, vc, table, cud, kvd.cpu()),
                 (q, kc, vc, table.t().contiguous().t(), cud, kvd)):
        with pytest.raises(AvtHipError):
            ops.paged_attn(*args)
    with pytest.raises(AvtHipError, match='out'):
        ops.paged_attn(q, kc, vc, table, cud, kvd, out=torch.empty((5, 255), device='cuda', dtype=BF16))
    for P, page, hd in ((4, 24, 64), (4, 4, 64), (4, 16, 1032), (4, 16, 12)):
        c = torch.zeros((P, page, 1, hd), device='cuda', dtype=BF16)
        with pytest.raises(AvtHipError):
            ops.paged_attn(torch.zeros((2, 1, hd), device='cuda', dtype=BF16), c, c, i32([[0]]), i32([0, 2]), i32([5]))


def test_offsets_past_four_gib(ops):
    """A cache of 6 GiB: rows far behind 2^32 bytes are written and read back."""
    P, page, H, hd = 24576, 64, 4, 512
    kc, vc = (torch.empty((P, page, H, hd), device='cuda', dtype=BF16) for _ in range(2))
    g = torch.Generator(device='cuda').manual_seed(3)
    far = [P - 1, P - 2, 1, P - 3, 0, P - 4]
    k, v = (torch.randn((6 * page, H, hd), generator=g, device='cuda').to(BF16) for _ in range(2))
    slots = i32([far[i // page] * page + i % page for i in range(6 * page)])
    ops.paged_kv_write(k, v, kc, vc, slots)
    for i, pg in enumerate(far):
        assert torch.equal(kc[pg], k[i * page:(i + 1) * page]) and torch.equal(vc[pg], v[i * page:(i + 1) * page])
    q = torch.randn((70, H, hd), generator=g, device='cuda').to(BF16)
    out = ops.paged_attn(q, kc, vc, i32([far]), i32([0, 70]), i32([6 * page - 5]))
    ref, tol = attn_in_64(q, k.view(6, page, H, hd), v.view(6, page, H, hd), i32([[0, 1, 2, 3, 4, 5]]), [0, 70], [6 * page - 5], hd ** -0.5)
    assert float(((out.double() - ref).abs() - tol).max()) <= 0


# ---- 4-bit linear ------------------------------------------------------------------------------------------------------------------------------
def w4_in_64(x, w, bias, act, res):
    u = torch.stack([w.q & 15, w.q >> 4], dim=-1).view(w.N, w.K).double() - 8
    s = w.scales.double().repeat_interleave(w.group, 1)
    y = x.double() @ (u * s).t().contiguous()
    B = x.double().abs() @ ((u.abs() + 24) * s.abs()).t().contiguous()
    tol = w.K * 2.0 ** -23 * B
    if bias is not None:
        y = y + bias.double()
        tol = tol + 2.0 ** -23 * y.abs()
    if act:
        pre = y
        y = 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3)))
        tol = 1.13 * tol + 2.0 ** -18 * pre.abs()
    if res is not None:
        y = y + res.double()
    return y, tol + 2.0 ** -23 * y.abs() + 1e-30


@pytest.mark.parametrize('M,N,K,group', [(1, 2048, 2048, 128), (3, 100, 8192, 64), (1, 1, 32, 32), (2, 17, 96, 32), (16, 64, 192, 64), (17, 33, 256, 128), (5, 427, 1408, 128),
                                         (33, 1000, 512, 32), (64, 48, 1024, 64), (65, 50, 384, 128), (200, 130, 640, 32), (7, 15, 8192, 128), (4, 96, 10944, 64),
                                         (20, 12300, 256, 64), (21, 70, 384, 128), (36, 12300, 256, 128), (37, 6200, 160, 32), (48, 6200, 256, 128)])
@pytest.mark.parametrize('epi', ['plain', 'bias', 'gelu', 'res', 'all', 'f32'])
def test_w4_linear_against_64_bits(ops, M, N, K, group, epi):
    g = torch.Generator(device='cuda').manual_seed(M * 1000 + N + K)
    x = (torch.randn((M, K + 8), generator=g, device='cuda') + 0.25).to(BF16)[:, :K]
    w = ops.W4Weight(torch.randint(0, 256, (N, K // 2), generator=g, device='cuda', dtype=torch.uint8), (torch.rand((N, K // group), generator=g, device='cuda') * 0.02 - 0.005).to(BF16))
    bias = torch.randn(N, generator=g, device='cuda') if epi in ('bias', 'all', 'gelu') else None
    res = torch.randn((M, N + 3), generator=g, device='cuda').to(BF16)[:, :N] if epi in ('res', 'all') else None
    act = ops.ACT_GELU_TANH if epi in ('gelu', 'all') else ops.ACT_NONE
    mode = ops.OUT_F32 if epi == 'f32' else ops.OUT_BF16
    big = torch.full((M, N + 5), 7.0, device='cuda', dtype=torch.float32 if epi == 'f32' else BF16)
    y = ops.w4_linear(x, w, bias=bias, act=act, res=res, out_mode=mode, out=big[:, :N])
    assert bool((big[:, N:] == 7.0).all())
    ref, tol = w4_in_64(x, w, bias, act, res)
    if epi != 'f32':
        tol = tol + U * ref.abs()
    assert float(((y.double() - ref).abs() - tol).max()) <= 0, float((y.double() - ref).abs().max())


def test_w4_special_values(ops):
    """A scale of zero, a row of x that is not finite: only its own outputs."""
    w = ops.W4Weight(torch.randint(0, 256, (40, 64), device='cuda', dtype=torch.uint8), torch.ones((40, 1), device='cuda', dtype=BF16))
    w.scales[3] = 0
    x = torch.ones((20, 128), device='cuda', dtype=BF16)
    x[5, 7] = float('nan')
    x[18, 100] = float('inf')
    y = ops.w4_linear(x, w)
    ok = [i for i in range(20) if i not in (5, 18)]
    assert bool(torch.isfinite(y[ok]).all()) and bool(torch.isnan(y[5]).all()) and not y[ok, 3].any()
    assert not bool(torch.isfinite(y[18]).all())


@pytest.mark.parametrize('group', [32, 64, 128])
def test_w4_quantize_is_the_nearest(ops, group):
    g = torch.Generator(device='cuda').manual_seed(group)
    wf = torch.randn((50, 384), generator=g, device='cuda') * 0.05
    wf[7] = 0
    w = ops.W4Weight.quantize(wf, group)
    step = w.scales.float().repeat_interleave(group, 1)
    assert bool(((w.dequantize() - wf).abs() <= 0.5 * step * (1 + 2.0 ** -6) + 7 * step * 2.0 ** -8).all())      # half a step; the largest also carries the scale's own rounding
    assert not w.dequantize()[7].any()


def test_w4_refuses_and_takes_nothing(ops):
    w = ops.W4Weight(torch.zeros((8, 64), device='cuda', dtype=torch.uint8), torch.zeros((8, 1), device='cuda', dtype=BF16))
    x = torch.zeros((2, 128), device='cuda', dtype=BF16)
    assert ops.w4_linear(x[:0], w).shape == (0, 8)
    for kw in (dict(bias=torch.zeros(7, device='cuda')), dict(res=torch.zeros((2, 7), device='cuda', dtype=BF16)), dict(act=ops.ACT_GELU_ERF), dict(out_mode=ops.OUT_ACCUM_F32),
               dict(out=torch.zeros((2, 8), device='cuda')), dict(bias=torch.zeros(8))):
        with pytest.raises(AvtHipError):
            ops.w4_linear(x, w, **kw)
    for bad in (x.float(), x[:, :64], x.cpu(), torch.zeros((2, 132), device='cuda', dtype=BF16)[:, 4:]):
        with pytest.raises(AvtHipError):
            ops.w4_linear(bad, w)
    for q, s in ((torch.zeros((8, 64), dtype=torch.uint8), torch.zeros((8, 3), dtype=BF16)), (torch.zeros((8, 64), dtype=torch.int8), torch.zeros((8, 1), dtype=BF16)),
                 (torch.zeros((8, 64), dtype=torch.uint8), torch.zeros((8, 1))), (torch.zeros((8, 256), dtype=torch.uint8), torch.zeros((8, 2), dtype=BF16))):
        with pytest.raises(AvtHipError):
            ops.W4Weight(q.cuda(), s.cuda())


# ---- a run of them together: the head's streams ------------------------------------------------------------------------------------------------
def build_head(in_dim, inter, layers, heads, seed=0):
    """(the head on the GPU, the oracle's with the same weights)."""
    from helpers import build_hip_model, build_oracle_model
    torch.manual_seed(seed)
    orc = build_oracle_model('feat', in_dim, inter, layers, heads, 11).future_predictor
    with torch.no_grad():
        for p in orc.parameters():
            if p.ndim >= 2:
                p.normal_(0, 0.6 * p.size(-1) ** -0.5)
    model = build_hip_model('feat', in_dim, inter, layers, heads, 11).eval()
    model.future_predictor.load_state_dict(orc.state_dict())
    return model.future_predictor, orc.eval()


def oracle_decode(orc, clip, steps):
    """The oracle's decoded features of a clip (T, C) and of a roll-out of `steps` from its end: (T - 1 + steps, C)."""
    with torch.no_grad():
        orc.output_len = orc.output_len_eval = steps
        orc.avg_last_n, orc.return_past_too = -1, False
        past, future, _, _ = orc(clip[None], (1, steps, clip.size(1)))
    return torch.cat([past[0, 1:], future[0]], 0)


TOL = 3e-2      # of the largest magnitude: the head's own limit against the fp32 oracle (bf16 activations and weights in every product)


def close(a, b):
    a, b = a.detach().double().cpu(), b.detach().double().cpu()
    assert float((a - b).abs().max()) <= TOL * float(b.abs().max()), float((a - b).abs().max() / b.abs().max())


@pytest.mark.parametrize('in_dim,inter,layers,heads,page', [(64, 64, 2, 2, 8), (128, 256, 2, 1, 16), (768, 2048, 6, 4, 16)])
def test_streams_of_different_lengths_match_the_oracle(ops, in_dim, inter, layers, heads, page):
    """Frames come in chunks of every size; each stream decodes what the oracle decodes of its clip alone, and rolls out as it does."""
    head, orc = build_head(in_dim, inter, layers, heads)
    g = torch.Generator().manual_seed(1)
    total = [5, 0, 20, 13, 1]
    clips = [torch.randn((t, in_dim), generator=g) for t in total]
    st = head.open_streams(5, max_len=30, page=page)
    seen, got = [0] * 5, [[] for _ in range(5)]
    for counts in ([2, 0, 11, 1, 0], [0, 0, 0, 0, 0], [1, 0, 8, 9, 0], [2, 0, 1, 3, 1]):
        feats = torch.cat([c[s:s + n] for c, s, n in zip(clips, seen, counts)])
        out = st.append(feats.cuda(), counts)
        for s, part in enumerate(out.split(counts)):
            got[s].append(part)
        seen = [a + b for a, b in zip(seen, counts)]
    assert st.lengths == total == seen
    fut = st.rollout(4)
    again = st.rollout(4)                                      # the streams are as they were
    assert torch.equal(fut, again) and not fut[1].any()
    for s, t in enumerate(total):
        if t:
            want = oracle_decode(orc, clips[s], 4)
            close(torch.cat(got[s]), want[:t])
            close(fut[s], want[t - 1:])
    more = torch.randn((3, in_dim), generator=g)               # and go on from their frames, not from what was rolled out
    out = st.append(more.cuda(), [3, 0, 0, 0, 0])
    close(out, oracle_decode(orc, torch.cat([clips[0], more]), 1)[5:])


def test_streams_release_and_refuse(ops):
    head, orc = build_head(64, 64, 2, 2)
    st = head.open_streams(3, max_len=40, page=8, pages=7)
    g = torch.Generator().manual_seed(2)
    x = torch.randn((40, 64), generator=g)
    first = st.append(x[:30].cuda(), [20, 10, 0])              # 3 + 2 pages
    with pytest.raises(ValueError, match='pages short'):
        st.append(x[:17].cuda(), [0, 0, 17])                   # 3 more: 2 are there
    with pytest.raises(ValueError, match='more than its 40'):
        st.append(x[:21].cuda(), [21, 0, 0])
    with pytest.raises(ValueError, match='more than its 40'):
        st.rollout(22)
    for feats, counts in ((x[:3].cuda(), [1, 1]), (x[:3].cuda(), [1, 1, 2]), (x[:3].cuda(), [4, -1, 0]), (x[:3, :32].cuda(), [1, 1, 1])):
        with pytest.raises(ValueError):
            st.append(feats, counts)
    assert st.lengths == [20, 10, 0]                           # what was refused left nothing behind
    st.release([0, 0])
    assert st.lengths == [0, 10, 0] and int(st.n_free) == 5
    out = st.append(torch.cat([x[:17], x[20:21]]).cuda(), [17, 1, 0])      # stream 0 is another clip now, on used pages
    close(out[:17], oracle_decode(orc, x[:17], 1))
    close(out[17:], oracle_decode(orc, torch.cat([x[20:30], x[20:21]]), 1)[10:])
    close(out[:17], first[:17])
    for kw in (dict(page=12), dict(max_len=0), dict(max_len=5000), dict(weight_bits=8), dict(pages=0)):
        with pytest.raises(ValueError):
            head.open_streams(2, **kw)


def test_streams_release_of_what_is_not_there(ops):
    """Refused as a whole: a number that is no stream (a negative one would count from the end) leaves every stream and page where it was."""
    head, orc = build_head(64, 64, 2, 2)
    st = head.open_streams(2, max_len=40, page=8, pages=7)
    x = torch.randn((20, 64), generator=torch.Generator().manual_seed(3))
    st.append(x[:15].cuda(), [9, 6])
    for which in ([0, 2], [-1], [1, 99]):
        with pytest.raises(ValueError, match='release'):
            st.release(which)
    assert st.lengths == [9, 6] and int(st.n_free) == 4
    out = st.append(x[15:17].cuda(), [1, 1])
    close(out[:1], oracle_decode(orc, torch.cat([x[:9], x[15:16]]), 1)[9:])
    close(out[1:], oracle_decode(orc, torch.cat([x[9:15], x[16:17]]), 1)[6:])


def test_streams_on_four_bit_weights(ops):
    """The same as a head whose projections hold the values that the 4-bit weights stand for."""
    head, _ = build_head(128, 256, 3, 2)
    st4 = head.open_streams(2, max_len=64, weight_bits=4)
    from avt_amd.models.streams import HeadStreams
    with torch.no_grad():
        for b in head.gpt_model.h:
            for lin in (b.attn.c_attn, b.attn.c_proj, b.mlp.c_fc, b.mlp.c_proj):
                lin.weight.copy_(HeadStreams._quantize(lin.weight).dequantize().t())
    st = head.open_streams(2, max_len=64)
    x = torch.randn((40, 128), generator=torch.Generator().manual_seed(4)).cuda()
    for lo, counts in ((0, [20, 5]), (25, [1, 1]), (27, [0, 13])):
        f = x[lo:lo + sum(counts)]
        close(st4.append(f, counts), st.append(f, counts))
    close(st4.rollout(3), st.rollout(3))


def test_streams_go_past_the_contiguous_cache_kernels_limits(ops):
    """A clip of 600 frames in chunks of 100 decodes as in one of 600 (the head's own attention takes 32 frames)."""
    head, _ = build_head(64, 128, 2, 2)
    x = torch.randn((600, 64), generator=torch.Generator().manual_seed(6)).cuda()
    a, b = head.open_streams(1), head.open_streams(1, page=64)
    parts = torch.cat([a.append(x[i:i + 100], [100]) for i in range(0, 600, 100)])
    close(parts, b.append(x, [600]))
    close(a.rollout(5), b.rollout(5))


# A row that sees a NaN has one, however the keys are split.  The hints give one split, a few (joined by the kernel of few splits) and many:
SPLIT_HINTS = [(100, 1), (250, 4), (1000, 10 ** 9)]             # (max_kv, the most splits it may give)


def splits_given(T, R, H, Hkv, hd, max_kv):
    """Partial results are hd + 2 floats a row and split, behind 16 bytes."""
    from avt_amd import lib
    return max(1, (lib.load().avt_paged_attn_workspace_bytes(T, R, H, Hkv, hd, 0, max_kv) - 16) // (4 * T * H * (hd + 2)))


@pytest.mark.parametrize('H,Hkv,hd', [(4, 4, 512), (8, 2, 128), (12, 12, 64), (4, 1, 256), (2, 2, 1024)])
@pytest.mark.parametrize('new', [1, 40])
@pytest.mark.parametrize('what', ['query', 'keys', 'value'])
def test_what_is_not_finite_and_seen_stays_however_the_keys_are_split(ops, H, Hkv, hd, new, what):
    """A query row with one NaN; 256 keys that are all NaN, whole splits of them; an infinite value among 256 keys whose probabilities are 0 in 32 bits (the sum of the
    definition is infinite): not finite in exactly those rows (for the value: that column), whatever max_kv says; every other row and column as the definition has it."""
    kv = 1000
    q, kc, vc, table, cu, kv_lens = make_attn([new, new], [kv, kv - 7], H, Hkv, hd, 16, 7 * hd + new)
    clean = (q.clone(), kc.clone(), vc.clone())
    T, grp = 2 * new, H // Hkv
    hit = torch.zeros((T, H, hd), dtype=torch.bool, device='cuda')
    put = lambda cache, lo, hi, head, col, x: [cache[int(table[0, j // 16]), j % 16, head, col].fill_(x) for j in range(lo, hi)]
    if what == 'query':
        q[0, H - 1, 3] = float('nan')
        hit[0, H - 1] = True
    elif what == 'keys':
        put(kc, 256, 512, Hkv - 1, slice(None), float('nan'))
        hit[:new, (Hkv - 1) * grp:] = True
    else:
        # q = 1 and k = -40 in every column: scale q k is -40 sqrt(hd), at most -320, below the others (random, |scale q k| < 20) by far more than 2^-149
        q[:new, H - 1] = 1.0
        put(kc, 256, 512, Hkv - 1, slice(None), -40.0)
        clean = (q.clone(), kc.clone(), vc.clone())
        put(vc, 300, 301, Hkv - 1, 5, float('inf'))
        hit[:new, (Hkv - 1) * grp:, 5] = True
        hit[:new, (Hkv - 1) * grp:H - 1, 5] = False            # (of the other rows with this kv head the probability may or may not be 0: not looked at)
    ref, tol = attn_in_64(*clean, table, cu, kv_lens, hd ** -0.5)
    look = ~hit
    if what == 'value':
        look[:new, (Hkv - 1) * grp:, 5] = False
    given = set()
    for max_kv, most in SPLIT_HINTS:
        n = splits_given(T, 2, H, Hkv, hd, max_kv)
        assert n <= most
        given.add(min(n, 5))
        out = ops.paged_attn(q, kc, vc, table, i32(cu), i32(kv_lens), max_kv=max_kv)
        o = out.view(T, H, hd)
        if what == 'value':
            assert not bool(torch.isfinite(o[hit]).any()), max_kv
        else:
            assert bool(torch.isnan(o[hit]).all()), max_kv
        ok = look.view(T, H * hd)
        assert bool(torch.isfinite(out[ok]).all()), max_kv
        assert float(((out.double() - ref).abs() - tol)[ok].max()) <= 0, max_kv
    assert 1 in given and len(given) > 1


@pytest.mark.parametrize('H,Hkv,hd', [(32, 1, 128), (64, 2, 64), (48, 1, 128), (64, 1, 40), (40, 1, 256), (32, 1, 512)])
@pytest.mark.parametrize('bad', [float('nan'), float('inf'), -float('inf')])
def test_many_query_heads_a_kv_head_and_what_a_row_does_not_see(ops, H, Hkv, hd, bad):
    """32 and more query heads share a kv head, so that all 32 rows of a wave may be one token's: the tile still holds keys of later tokens, for the other waves.  The
    last tokens' values (two of them, so that rows before, between and at them are there) are not finite: rows that do not see them are as if they were not there."""
    new, kv = [4, 70, 3, 33], [20, 100, 64, 300]
    q, kc, vc, table, cu, kv_lens = make_attn(new, kv, H, Hkv, hd, 16, 19)
    for r, k in enumerate(kv):
        for j in (k - 1, k - 2):
            vc[int(table[r, j // 16]), j % 16] = bad
    ref, tol = attn_in_64(q, kc, torch.nan_to_num(vc, 0, 0, 0), table, cu, kv_lens, hd ** -0.5)
    for kw in ({}, dict(max_new=70, max_kv=300), dict(max_new=1, max_kv=300)):
        out = ops.paged_attn(q, kc, vc, table, i32(cu), i32(kv_lens), **kw)
        for r in range(len(new)):
            lo, hi = cu[r], cu[r + 1] - 2
            assert bool(torch.isfinite(out[lo:hi]).all()), (r, kw)
            assert float(((out[lo:hi].double() - ref[lo:hi]).abs() - tol[lo:hi]).max()) <= 0
            assert not bool(torch.isfinite(out[hi:cu[r + 1]]).any())                # and what IS seen is passed on


@pytest.mark.parametrize('bits', [16, 4])
def test_a_rollout_keeps_no_page(ops, bits):
    """A pool that holds the frames and little more: what a roll-out took on its way is free again, and another stream may have it."""
    head, orc = build_head(64, 64, 2, 2)
    st = head.open_streams(3, max_len=40, page=8, pages=6, weight_bits=bits)
    x = torch.randn((48, 64), generator=torch.Generator().manual_seed(8))
    st.append(x[:15].cuda(), [8, 7, 0])                        # 1 + 1 pages: 4 free
    state = lambda: (st.lens.tolist(), st.owned.tolist(), int(st.n_free), list(st._owned), st._n_free)
    before = state()
    assert before[2] == 4
    a = st.rollout(12)                                         # 11 frames behind each: 2 pages of stream 0, 2 of stream 1
    assert state() == before
    assert torch.equal(a, st.rollout(12)) and state() == before
    with pytest.raises(ValueError, match='pages short'):
        st.rollout(20)                                         # 3 + 3 pages: 4 are there
    assert state() == before
    out = st.append(x[15:47].cuda(), [0, 0, 32])               # all four free pages
    assert st.lengths == [8, 7, 32] and int(st.n_free) == 0
    if bits == 16:
        close(out, oracle_decode(orc, x[15:47], 1))
        close(a[0, :4], oracle_decode(orc, x[:8], 4)[7:])
    b = st.rollout(1)              # (a step more would need a page of stream 0)
    assert torch.equal(b[:2], a[:2, :1])
    out = st.append(x[47:48].cuda(), [0, 1, 0])                # stream 1's own page has a row left, which the roll-outs wrote over
    if bits == 16:
        close(out, oracle_decode(orc, torch.cat([x[8:15], x[47:48]]), 1)[7:])


def test_an_append_that_fails_leaves_the_streams_as_they_were(ops, monkeypatch):
    """Features on another device, and an error on the way through the blocks: no page is taken, and the same frames may come again."""
    head, orc = build_head(64, 64, 2, 2)
    st = head.open_streams(2, max_len=40, page=8, pages=4)
    x = torch.randn((30, 64), generator=torch.Generator().manual_seed(9))
    st.append(x[:5].cuda(), [5, 0])
    state = lambda: (st.lens.tolist(), st.owned.tolist(), int(st.n_free), list(st._owned), st._n_free, st.lengths)
    before = state()
    with pytest.raises(ValueError, match='device'):
        st.append(x[5:25], [20, 0])
    assert state() == before
    with monkeypatch.context() as m:
        calls = []

        def broken(*a, **kw):
            calls.append(1)
            if len(calls) > 2:
                raise RuntimeError('out of memory')
            return ops_ln(*a, **kw)
        ops_ln = ops.layernorm_fwd
        m.setattr(ops, 'layernorm_fwd', broken)
        with pytest.raises(RuntimeError, match='out of memory'):
            st.append(x[5:25].cuda(), [20, 0])
        calls.clear()
        with pytest.raises(RuntimeError, match='out of memory'):
            st.rollout(9)
    assert state() == before
    out = st.append(x[5:29].cuda(), [3, 21])                   # three pages for stream 1: all four are in use
    close(out[:3], oracle_decode(orc, x[:8], 1)[5:])
    close(out[3:], oracle_decode(orc, x[8:29], 1))


# ---- 4-bit linear: sums that are exact --------------------------------------------------------------------------------------------------------
def w4_exact_case(M, N, K, group, seed):
    """Inputs whose every partial sum, in any order, is a whole number of 2^-7 below 2^24 of them, i.e. exact in fp32: x in -2 .. 2, scales of 8 significant bits
    c 2^-7 with odd c in 129 .. 255 (a weight (u - 8) s has up to 11 bits and would not survive a rounding to bf16), bias and residual whole numbers.
    Returns CPU tensors (x, q bytes, scales, bias, res, exact) with exact int64 in units of 2^-7."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randint(-2, 3, (M, K), generator=g)
    q = torch.randint(0, 256, (N, K // 2), generator=g, dtype=torch.uint8)
    c = 2 * torch.randint(64, 128, (N, K // group), generator=g) + 1
    bias, res = torch.randint(-9, 10, (N,), generator=g), torch.randint(-9, 10, (M, N), generator=g)
    total, bound = torch.zeros((M, N), dtype=torch.int64), torch.zeros((M, N), dtype=torch.int64)
    for i in range(K // group):                                # (products of whole numbers in fp64: exact)
        b = q[:, i * group // 2:(i + 1) * group // 2]
        xs, us = x[:, i * group:(i + 1) * group].double(), torch.stack([b & 15, b >> 4], dim=-1).view(N, group).double()
        part = (xs @ (us - 8).t()).long() * c[:, i]
        total += part
        bound += part.abs()
        assert int((xs.abs() @ (us + 16).t()).max()) < 1 << 24                       # inside a group: products of 16 + u, and 24 sum x
    assert int(bound.max()) + 9 * 128 * 2 < 1 << 24
    return x, q, c, bias, res, total


def w4_case_on_gpu(ops, x, q, c, bias, res):
    K = x.size(1)
    wide = torch.zeros((x.size(0), K + 8), device='cuda', dtype=BF16)
    wide[:, :K] = x.cuda()
    return wide[:, :K], ops.W4Weight(q.cuda(), (c.cuda().double() / 128).to(BF16)), bias.float().cuda(), res.cuda().to(BF16)


W4_EXACT = [(1, 2048, 2048, 128), (3, 100, 8192, 64), (7, 15, 8192, 128), (4, 96, 10944, 64), (2, 17, 96, 32), (16, 64, 192, 64), (17, 33, 256, 128), (33, 1000, 544, 32),
            (64, 2048, 2048, 64), (64, 48, 8192, 32), (36, 12300, 1376, 32), (48, 6200, 4160, 64), (20, 12300, 1152, 128), (33, 12300, 8192, 128), (65, 50, 10944, 32), (200, 130, 8192, 128)]


@pytest.mark.parametrize('M,N,K,group', W4_EXACT)
def test_w4_linear_of_exact_sums_is_exact(ops, M, N, K, group):
    """Every weight, scale and group counts once, unrounded: equal, in fp32, with and without bias and residual."""
    x, q, c, bias, res, total = w4_exact_case(M, N, K, group, M + N + K)
    xd, w, bd, rd = w4_case_on_gpu(ops, x, q, c, bias, res)
    y = ops.w4_linear(xd, w, out_mode=ops.OUT_F32)
    assert torch.equal(y.double().cpu() * 128, total.double())
    y = ops.w4_linear(xd, w, bias=bd, res=rd, out_mode=ops.OUT_F32)
    assert torch.equal(y.double().cpu() * 128, (total + 128 * (bias + res)).double())
    y = ops.w4_linear(xd, w)                                   # and rounded once
    assert torch.equal(y.cpu(), (total.double() / 128).float().to(BF16))


@pytest.mark.parametrize('counts', [[1] * 64, [90, 0, 200, 1, 37]])
def test_four_bit_streams_of_many_rows(ops, counts):
    """64 streams of one frame each, and chunks of hundreds of rows: the same as a head whose projections hold the values that the 4-bit weights stand for."""
    from avt_amd.models.streams import HeadStreams
    head, _ = build_head(128, 256, 2, 2)
    st4 = head.open_streams(len(counts), max_len=300, weight_bits=4)
    with torch.no_grad():
        for b in head.gpt_model.h:
            for lin in (b.attn.c_attn, b.attn.c_proj, b.mlp.c_fc, b.mlp.c_proj):
                lin.weight.copy_(HeadStreams._quantize(lin.weight).dequantize().t())
    st = head.open_streams(len(counts), max_len=300)
    x = torch.randn((2, sum(counts), 128), generator=torch.Generator().manual_seed(5)).cuda()
    for f in x[:2 if max(counts) < 100 else 1]:
        close(st4.append(f, counts), st.append(f, counts))
    close(st4.rollout(2), st.rollout(2))
