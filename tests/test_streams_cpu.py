"""CPU (-m "not gpu"): what the streams' operators refuse on the host, before any launch, and the parts of them that are host work."""
import pytest
import torch

from avt_amd import lib, ops
from avt_amd.lib import AvtHipError

BF16, I32 = torch.bfloat16, torch.int32
P = 1 << 20                     # an aligned address that nothing reads: every call below is refused before a launch


def plan(**kw):
    a = dict(lens=P, fresh=P, owned=P, table=P, ldt=4, width=4, free=P, nfree=8, n_free=P, page=16, R=2, T=3, cu=P, kv=P, own=P, nf=P, slots=P, pos=P, st=P)
    a.update(kw)
    lib.call('avt_paged_plan', *a.values(), None)


@pytest.mark.parametrize('kw,match', [(dict(lens=None), 'null'), (dict(free=None), 'free list'), (dict(slots=None), 'token output'), (dict(R=0), 'streams'), (dict(R=4097), 'streams'),
                                      (dict(T=-1), 'sizes'), (dict(width=0), 'sizes'), (dict(ldt=3), 'sizes'), (dict(nfree=-1), 'sizes'), (dict(page=0), 'page'), (dict(page=24), 'page'),
                                      (dict(page=4), 'page'), (dict(page=2048), 'page'), (dict(width=1 << 22, ldt=1 << 22, page=1024), '2\\^31')])
def test_plan_refusals(kw, match):
    with pytest.raises(AvtHipError, match=match):
        plan(**kw)


def write(**kw):
    a = dict(k=P, ldk=128, v=P, ldv=128, kc=P, vc=P, slots=P, nslots=64, T=3, width=128)
    a.update(kw)
    lib.call('avt_paged_kv_write', *a.values(), None)


@pytest.mark.parametrize('kw,match', [(dict(k=None), 'null'), (dict(slots=None), 'null'), (dict(width=12), 'multiple of 8'), (dict(width=0), 'multiple of 8'), (dict(T=-1), 'multiple of 8'),
                                      (dict(ldk=120), '16-byte'), (dict(ldv=132), '16-byte'), (dict(k=P + 8), '16-byte'), (dict(vc=P + 2), '16-byte'), (dict(nslots=-1), 'null'),
                                      (dict(T=1 << 30, width=1 << 20, ldk=1 << 20, ldv=1 << 20), 'too many')])
def test_write_refusals(kw, match):
    with pytest.raises(AvtHipError, match=match):
        write(**kw)
    write(T=0, k=None)          # nothing to do is no error


def attn(**kw):
    a = dict(q=P, ldq=512, kc=P, vc=P, npages=4, page=16, table=P, ldt=4, width=4, cu=P, kv=P, out=P, ldo=512, T=3, R=2, H=4, Hkv=2, hd=128, scale=0.1, max_new=1, max_kv=64, ws=P, wsb=1 << 30)
    a.update(kw)
    lib.call('avt_paged_attn_fwd', *a.values(), None)


@pytest.mark.parametrize('kw,match', [(dict(q=None), 'null'), (dict(kv=None), 'null'), (dict(out=None), 'null'), (dict(H=3), 'sizes'), (dict(Hkv=0), 'sizes'), (dict(R=0), 'sizes'), (dict(T=-1), 'sizes'),
                                      (dict(hd=12), 'head_dim'), (dict(hd=0), 'head_dim'), (dict(hd=1032), 'head_dim'), (dict(page=40), 'page'), (dict(ldt=2), 'table'), (dict(width=0), 'table'),
                                      (dict(npages=-1), 'table'), (dict(ldq=504), '16-byte'), (dict(ldo=508), '16-byte'), (dict(kc=P + 4), '16-byte'), (dict(Hkv=1 << 20, H=1 << 20, ldq=1 << 30, ldo=1 << 30), 'too long'), (dict(ldq=1 << 29), 'too far'),
                                      (dict(width=1 << 21, ldt=1 << 21, page=1024), 'table'),
                                      (dict(T=1 << 29, H=8, ldq=1024, ldo=1024), 'too many'), (dict(ws=None, max_kv=100000, width=8192, ldt=8192), 'workspace'),
                                      (dict(wsb=16, max_kv=100000, width=8192, ldt=8192), 'workspace')])
def test_attention_refusals(kw, match):
    with pytest.raises(AvtHipError, match=match):
        attn(**kw)
    attn(T=0, q=None)


def test_attention_workspace_grows_with_the_splits_and_never_overflows():
    q = lib.load().avt_paged_attn_workspace_bytes
    assert q(1, 1, 4, 4, 512, 1, 100) == 16                                     # one split: nothing
    assert q(1, 1, 4, 4, 512, 1, 100000) >= 4 * 100 * 4 * 514                   # a long stream alone on the chip: many
    assert q(4096, 1, 8, 8, 64, 4096, 0) >= 16 and q(0, 1, 1, 1, 1, 0, 0) == 16
    assert q(1 << 20, 1, 64, 64, 128, 1 << 20, 2 ** 31 - 1) < 1 << 50


def w4(**kw):
    a = dict(x=P, ldx=256, q=P, s=P, group=64, bias=None, act=0, res=None, ldres=0, out=P, ldo=32, mode=0, M=2, N=32, K=256)
    a.update(kw)
    lib.call('avt_w4_linear', *a.values(), None)


@pytest.mark.parametrize('kw,match', [(dict(x=None), 'null'), (dict(s=None), 'null'), (dict(group=16), 'group'), (dict(group=0), 'group'), (dict(K=224, group=64), 'multiple of the group'), (dict(act=1), 'act'),
                                      (dict(act=3), 'act'), (dict(mode=2), 'out_mode'), (dict(M=-1), 'sizes'), (dict(N=0), 'sizes'), (dict(K=0), 'sizes'), (dict(ldx=248), '16-byte'), (dict(ldx=260), '16-byte'),
                                      (dict(x=P + 8), '16-byte'), (dict(q=P + 4), '16-byte'), (dict(ldo=31), 'leading dimension'), (dict(res=P, ldres=31), 'leading dimension'),
                                      (dict(K=1 << 25, ldx=1 << 25), '2\\^24'), (dict(M=1 << 27), 'too many')])
def test_w4_refusals(kw, match):
    with pytest.raises(AvtHipError, match=match):
        w4(**kw)
    w4(M=0, x=None)


def test_the_wrappers_refuse_cpu_tensors_and_wrong_shapes():
    i = lambda *v: torch.tensor(v, dtype=I32)
    with pytest.raises(AvtHipError, match='GPU'):
        ops.paged_plan(i(1), i(1), i(1), i(0).view(1, 1), i(0), i(1), 16, 1)
    with pytest.raises(AvtHipError, match='new'):
        ops.paged_plan(i(1), i(1, 2), i(1), i(0).view(1, 1), i(0), i(1), 16, 1)
    with pytest.raises(AvtHipError, match='table'):
        ops.paged_plan(i(1), i(1), i(1), i(0), i(0), i(1), 16, 1)
    c, q = torch.zeros((2, 16, 2, 64), dtype=BF16), torch.zeros((3, 4, 64), dtype=BF16)
    with pytest.raises(AvtHipError, match='GPU'):
        ops.paged_kv_write(q[:, :2], q[:, 2:], c, c.clone(), i(0, 1, 2))
    with pytest.raises(AvtHipError, match='rows'):
        ops.paged_kv_write(q, q, c, c.clone(), i(0, 1, 2))
    with pytest.raises(AvtHipError, match='GPU'):
        ops.paged_attn(q, c, c.clone(), i(0).view(1, 1), i(0, 3), i(3))
    with pytest.raises(AvtHipError, match='multiple of 2 heads'):
        ops.paged_attn(q[:, :3], c, c.clone(), i(0).view(1, 1), i(0, 3), i(3))
    with pytest.raises(AvtHipError, match='cu'):
        ops.paged_attn(q, c, c.clone(), i(0).view(1, 1), i(0, 3, 3), i(3))
    w = ops.W4Weight(torch.zeros((8, 64), dtype=torch.uint8), torch.zeros((8, 1), dtype=BF16))
    with pytest.raises(AvtHipError, match='GPU'):
        ops.w4_linear(torch.zeros((1, 128), dtype=BF16), w)
    with pytest.raises(AvtHipError, match='x must be'):
        ops.w4_linear(torch.zeros((1, 64), dtype=BF16), w)


def test_w4_layout_and_rounding():
    """Two values to a byte, the even k in the low nibble; the nearest of the 16 steps of the stored scale."""
    w = torch.zeros((1, 32))
    w[0, :4] = torch.tensor([7.0, -7.0, 1.0, -0.4])
    p = ops.W4Weight.quantize(w, 32)
    assert p.scales.item() == 1.0 and p.q[0, 0] == (15 | 1 << 4) and p.q[0, 1] == (9 | 8 << 4) and p.q[0, 2] == (8 | 8 << 4)
    assert torch.equal(p.dequantize(), w.round())
    g = torch.Generator().manual_seed(0)
    w = torch.randn((9, 256), generator=g)
    for group in (32, 64, 128):
        p = ops.W4Weight.quantize(w, group)
        assert (p.N, p.K, p.group) == (9, 256, group)
        s = p.scales.float().repeat_interleave(group, 1)
        # half a step, and for the largest values what the scale's own rounding (half a step of bf16, 2^-8) takes off seven steps
        assert bool(((p.dequantize() - w).abs() <= s * (0.5 + 7 * 2.0 ** -8) * (1 + 2.0 ** -20)).all())
    with pytest.raises(AvtHipError):
        ops.W4Weight.quantize(w, 48)


def test_open_streams_refuses_what_its_operators_would():
    """Before anything is allocated: more streams than a plan takes, heads wider than the attention's, a pool whose rows no slot could name."""
    from helpers import build_hip_model
    head = build_hip_model('feat', 64, 64, 1, 2, 11, device='cpu').future_predictor
    for kw, match in ((dict(streams=4097), '4096'), (dict(streams=2, pages=1 << 28, page=16), '2\\^31'), (dict(streams=0), 'at least one'), (dict(streams=1, page=12), 'page')):
        with pytest.raises(ValueError, match=match):
            head.open_streams(**kw)
    wide = build_hip_model('feat', 64, 1032, 1, 1, 11, device='cpu').future_predictor
    with pytest.raises(ValueError, match='1024'):
        wide.open_streams(2)


def test_caches_of_more_rows_than_a_slot_can_name_are_refused():
    """A slot is an int32: the plan gives rows behind 2^31 - 1 none, so an attention that saw them would see keys that were never written."""
    with pytest.raises(AvtHipError, match='2\\^31'):
        attn(npages=(1 << 27) + 1, page=16)
    with pytest.raises(AvtHipError, match='2\\^31'):
        attn(npages=1 << 60, page=1024)
    attn(T=0, q=None, npages=1 << 27, page=16)
    with pytest.raises(AvtHipError, match='2\\^31'):
        write(nslots=(1 << 31) + 1)
    write(T=0, k=None, nslots=1 << 31)


@pytest.mark.parametrize('M,N,K,group', [(3, 40, 8192, 64), (4, 96, 10944, 64), (2, 40, 10944, 32)])
def test_exact_sums_tell_every_mistake(M, N, K, group):
    """The inputs of the GPU's test of equality, with mistakes planted in the sums: a group left out, first, last or between, a neighbour's scale, weights
    rounded to bf16, a piece of 32 k left out.  Each moves most outputs (a sum of whole numbers is 0 by chance once in some ten)."""
    import test_streams_gpu as t
    x, q, c, _, _, total = t.w4_exact_case(M, N, K, group, M + N + K)
    u = torch.stack([q & 15, q >> 4], dim=-1).view(N, K).double() - 8
    s = c.double().repeat_interleave(group, 1)
    xs, full = x.double(), total.double()
    assert torch.equal(xs @ (u * s).t(), full)
    moved = lambda y: float((y != full).double().mean())
    for lo, n in ((0, group), (K - group, group), (K // 2 // group * group, group), (K // 2 // 32 * 32, 32)):
        xz = xs.clone()
        xz[:, lo:lo + n] = 0
        assert moved(xz @ (u * s).t()) > 0.8
    s2 = s.clone()
    s2[:, -group:] = s[:, -2 * group:-group]
    assert moved(xs @ (u * s2).t()) > 0.8
    assert moved(xs @ (u * s).to(torch.bfloat16).double().t()) > 0.9


def test_plan_refuses_rows_that_its_threads_could_not_count():
    """A thread goes on by up to 512 x 1024 rows: from 2^31 - 2^20 rows on that could pass 2^31 and come out negative."""
    for T in (2 ** 31 - 1, 2 ** 31 - 2 ** 19, 2 ** 31 - 2 ** 20):
        with pytest.raises(AvtHipError, match='2\\^31 - 2\\^20'):
            plan(T=T)
