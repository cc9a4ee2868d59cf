"""CPU (-m "not gpu"): host logic of the product -- C-ABI library loads and exports every symbol include/avt_hip.h
declares, the config shim composes the reference-style YAML, modules keep the reference's state_dict names, LR
schedulers reproduce the reference sequence, the product path refuses CPU tensors, and the gradient reducer is correct
across 2 gloo ranks."""
import os
import re
import subprocess
import sys

import numpy as np
import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_abi_library_exports_every_declared_symbol():
    from avt_amd import lib
    header = open(os.path.join(ROOT, 'include', 'avt_hip.h')).read()
    declared = set(re.findall(r'^(?:int|size_t|const char\*)\s+(avt_\w+)\s*\(', header, flags=re.M))
    assert declared, 'no declarations parsed'
    bound = set(lib.SIGNATURES) | set(lib.SIZE_QUERIES) | {'avt_last_error'}
    assert declared == bound, declared ^ bound
    l = lib.load()                       # dlopen; getattr on every symbol; ABI version check
    for name in declared:
        assert hasattr(l, name), name
    assert l.avt_abi_version() == lib.ABI_VERSION
    # argument counts in the binding match the header
    for name in lib.SIGNATURES:
        m = re.search(r'int\s+' + name + r'\s*\((.*?)\);', header, flags=re.S)
        args = [a for a in m.group(1).split(',') if a.strip() and a.strip() != 'void']
        assert len(args) == len(lib.SIGNATURES[name]), (name, len(args), len(lib.SIGNATURES[name]))
    for name in lib.SIZE_QUERIES:
        m = re.search(r'size_t\s+' + name + r'\s*\((.*?)\);', header, flags=re.S)
        args = [a for a in m.group(1).split(',') if a.strip() and a.strip() != 'void']
        assert len(args) == len(lib.SIZE_QUERIES[name]), (name, len(args))
        assert getattr(l, name)(*([64] * len(args))) > 0
    # ... and nothing but the declared C symbols leaves the library (csrc/exports.map): no mangled internals, no toolchain markers
    nm = subprocess.run(['nm', '-D', '--defined-only', lib.LIB_PATH], capture_output=True, text=True, check=True).stdout
    exported = {ln.split()[-1] for ln in nm.splitlines() if ln.strip()}
    assert exported == declared | {'avt_abi_version'} or exported == declared, exported ^ declared


def test_host_side_validation_rejects_bad_calls_without_a_gpu():
    """Shape/alignment violations are rejected on the host before any launch (no GPU needed to see the error)."""
    from avt_amd import lib
    with pytest.raises(lib.AvtHipError, match='null operand'):
        lib.call('avt_gemm_bf16', None, 1, 8, None, 1, 8, None, 8, 8, 8, 8, None, 0, None, 0, None, 0, None, 0, 0, 0.0, 0, None, 0, 0, 0, None, 0, None)
    with pytest.raises(lib.AvtHipError, match='head_dim must be 64'):
        lib.call('avt_vit_attn_fwd', 16, 16, 16, 1, 5, 1, 32, 0.125, None)
    with pytest.raises(lib.AvtHipError, match='multiple of 8'):
        lib.call('avt_layernorm_fwd', 16, 12, 16, 16, 16, 12, None, None, 4, 12, 1e-6, None)


def test_product_ops_refuse_cpu_tensors():
    from avt_amd import ops
    from avt_amd.lib import AvtHipError
    a = torch.zeros((8, 8), dtype=torch.bfloat16)
    with pytest.raises(AvtHipError, match='no CPU fallback'):
        ops.gemm(a, a, 8, 8, 8)


def test_config_compose_matches_reference_experiment_keys():
    from avt_amd.config import compose, read_overrides
    cfg = compose(os.path.join(ROOT, 'conf'), read_overrides(os.path.join(ROOT, 'expts', '01_ek100_avt.txt')))
    assert cfg.model.backbone._target_ == 'models.video_classification.TIMMModel'
    assert cfg.model.backbone.model_type == 'vit_base_patch16_224_in21k'
    assert cfg.model.future_predictor == {'_target_': 'models.future_prediction.AVTh', 'n_head': 4, 'n_layer': 6, 'output_len': 1,
                                          'inter_dim': 2048, 'return_past_too': True, 'future_pred_loss': {'_target_': 'torch.nn.MSELoss'},
                                          'future_pred_loss_wt': 1.0, 'avg_last_n': 1}
    assert cfg.opt.optimizer == {'_target_': 'torch.optim.SGD', 'momentum': 0.9, 'nesterov': True}
    assert cfg.opt.lr_wd == [['__all__', 0.0001, 1e-06]]
    assert cfg.opt.scheduler.num_epochs == 30 and cfg.opt.warmup.num_epochs == 20
    assert cfg.data_train.num_frames == 10 and cfg.data_eval.num_frames == 10 and cfg.data_train.subclips.num_frames == 1
    assert cfg.train.train_one_epoch_fn.loss_wts.feat == 1.0 and cfg.train.train_one_epoch_fn.loss_wts.past_cls_action == 1.0
    assert cfg.model.dropout == 0.2 and cfg.model.classifier_on_past is True
    cfg7 = compose(os.path.join(ROOT, 'conf'), read_overrides(os.path.join(ROOT, 'expts', '07_ek100_avt_longer.txt')))
    assert cfg7.data_train.num_frames == 15
    # resolvers (train_net.py:17-19)
    cfg2 = compose(os.path.join(ROOT, 'conf'), ['train.num_epochs=45', 'opt.warmup.num_epochs=5'])
    assert cfg2.opt.scheduler.num_epochs == 40


def test_modules_keep_reference_state_dict_names_and_shapes():
    """Checkpoint compatibility: identical names/shapes to the oracle, which mirrors timm / HF / reference."""
    from helpers import build_oracle_model
    from avt_amd.config import compose, instantiate, read_overrides
    from avt_amd.models.base_model import BaseModel
    cfg = compose(os.path.join(ROOT, 'conf'), read_overrides(os.path.join(ROOT, 'expts', '01_ek100_avt.txt')))
    model = BaseModel(cfg.model, {'action': 3806}, {})
    orc = build_oracle_model('vit', 768, 2048, 6, 4, 3806, vit=(768, 12, 12, 224))
    a = {k: tuple(v.shape) for k, v in model.state_dict().items()}
    b = {k: tuple(v.shape) for k, v in orc.state_dict().items()}
    assert a == b
    assert sum(p.numel() for p in model.parameters()) == 396123358 or abs(sum(p.numel() for p in model.parameters()) - 396.12e6) < 0.01e6
    model.load_state_dict(orc.state_dict())             # round trip through the reference naming
    assert model.future_predictor.gpt_model.h[0].attn.c_attn.weight.shape == (2048, 6144)     # HF Conv1D (in, out)


def test_schedulers_reproduce_reference_lr_sequence(golden_dir):
    from avt_amd.common.scheduler import CosineLR, Warmup
    z = np.load(os.path.join(golden_dir, 'g4_lr_schedules.npz'))
    for key in z.files:
        W, C, I, B, N = [float(x[1:]) for x in key.split('_')]
        ref = z[key]

        class Opt:
            param_groups = [{'lr': B * N}]
        opt = Opt()
        cos = CosineLR(opt, num_epochs=int(C), iters_per_epoch=int(I), world_size=int(N), eta_min=0.0)
        wu = Warmup(opt, cos, init_lr_ratio=0.0, num_epochs=int(W), iters_per_epoch=int(I), world_size=int(N))
        lrs = []
        for _ in range(len(ref)):
            lrs.append(opt.param_groups[0]['lr'])
            wu.step()
        assert np.abs(np.asarray(lrs) - ref).max() < 1e-12, (key, lrs[:6], ref[:6])


def test_param_groups_follow_reference_rules():
    from avt_amd.func.train import _param_groups
    m = torch.nn.Sequential(torch.nn.Linear(4, 4), torch.nn.LayerNorm(4))
    groups = _param_groups(m, [['__all__', 0.1, 1e-3]], world_size=8, bias_bn_wd_scale=0.5)
    assert len(groups) == 2
    assert groups[0]['lr'] == pytest.approx(0.8) and groups[0]['weight_decay'] == 1e-3 and len(groups[0]['params']) == 2
    assert groups[1]['weight_decay'] == pytest.approx(5e-4) and len(groups[1]['params']) == 2
    assert _param_groups(m, [['__all__', 0.0, 0.0]], 1) == []


DDP_WORKER = r'''
import os, sys, torch, torch.distributed as dist
sys.path.insert(0, sys.argv[1])
from avt_amd.ddp import GradReducer
rank, world = int(os.environ['RANK']), int(os.environ['WORLD_SIZE'])
dist.init_process_group('gloo', init_method='env://', rank=rank, world_size=world)

class P:            # parameter stand-in
    pass
class Arena:        # CPU stand-in for avt_amd.arena.ParamArena: just the fields the reducer touches
    def __init__(self, sizes):
        self.params = [P() for _ in sizes]
        self.name_of = {id(p): i for i, p in enumerate(self.params)}
        self.offsets, off = {}, 0
        for i, s in enumerate(sizes):
            self.offsets[i] = off; off += s
        self.total = off
        self.grad = torch.zeros(off)
        self.master = torch.zeros(off)
    def refresh_shadow(self, force=False):
        pass
class Seg(torch.nn.Module):
    grad_ready_hook = None
    def forward(self, x):
        return x
class Model(torch.nn.Module):
    def __init__(self, arena):
        super().__init__(); self.segs = torch.nn.ModuleList([Seg(), Seg(), Seg()]); self._a = arena
    @property
    def arena(self):
        return self._a
sizes = [1000, 3000, 500, 2500, 800 + (len(sys.argv) > 4 and int(sys.argv[4]))]
arena = Arena(sizes)
model = Model(arena)
MODE, WIRE = sys.argv[2], (torch.bfloat16 if sys.argv[3] == 'bf16' else torch.float32)
red = GradReducer(model, bucket_bytes=4 * 1500, mode=MODE, wire_dtype=WIRE)
TOL = 1e-5 if WIRE == torch.float32 else 3e-2          # bf16 on the wire keeps 8 mantissa bits of every summand
close = lambda a, b: float((a - b).abs().max()) <= TOL * (1 + float(b.abs().max()))
arena.master.fill_(float(rank + 1)); GradReducer.broadcast_parameters(model)
assert float(arena.master[0]) == 1.0
torch.manual_seed(100 + rank)
g_local = torch.randn(arena.total)
gathered = [torch.zeros(arena.total) for _ in range(world)]
dist.all_gather(gathered, g_local)
expect = sum(gathered)
for step in range(2):
    red.start_step()
    arena.grad.copy_(g_local)
    # backward finishes segments from the END of the buffer: params 4,3 | 2,1 | 0
    model.segs[2].grad_ready_hook(arena.params[3], arena.params[4])
    model.segs[1].grad_ready_hook(arena.params[1], arena.params[2])
    model.segs[0].grad_ready_hook(arena.params[0], arena.params[0])
    red.finish()
    assert close(arena.grad, expect), float((arena.grad - expect).abs().max())
    st = red.stats()
    assert st['buckets_per_step'] == red.launched >= 5 and st['mode'] == MODE, st       # 7800 elements in 1500-element buckets
    assert st['bytes_per_step'] == arena.total * (4 if WIRE == torch.float32 else 2), st
# no hook fired at all -> finish() still reduces everything
red.start_step(); arena.grad.copy_(g_local); red.finish()
assert close(arena.grad, expect) and red.launched == 1
# a module that ran forward twice this step (multi-crop clips: one fused node per crop, models/base_model.py:251-273): its
# range may only be handed to the collective after the SECOND backward, which keeps accumulating into it
red.start_step()
model.segs[2](torch.zeros(1)); model.segs[2](torch.zeros(1))     # the reducer counts forwards itself (forward pre-hook)
with torch.no_grad():
    model.segs[1](torch.zeros(1)); model.segs[1](torch.zeros(1))          # evaluation passes do not count
model.segs[1](torch.zeros(1))
arena.grad.zero_()
arena.grad[arena.offsets[3]:].add_(g_local[arena.offsets[3]:] * 0.25)         # first crop's contribution
model.segs[2].grad_ready_hook(arena.params[3], arena.params[4])
assert red._lo == arena.total, 'range released after the first of two backwards'
arena.grad[arena.offsets[3]:].add_(g_local[arena.offsets[3]:] * 0.75)         # second crop
model.segs[2].grad_ready_hook(arena.params[3], arena.params[4])
assert red._lo == arena.offsets[3]
arena.grad[:arena.offsets[3]].copy_(g_local[:arena.offsets[3]])
model.segs[1].grad_ready_hook(arena.params[1], arena.params[2])
model.segs[0].grad_ready_hook(arena.params[0], arena.params[0])
red.finish()
assert close(arena.grad, expect), float((arena.grad - expect).abs().max())
# the tail rule: once the not-yet-produced head of the buffer is at most tail_bytes, everything produced so far is sent at once, so
# that finish() -- the only exchange backward cannot hide -- has just that head left; and a paused reducer exchanges nothing
red2 = GradReducer(model, bucket_bytes=4 * 1500, mode=MODE, wire_dtype=WIRE, tail_bytes=4 * 1200)
red2.start_step(); arena.grad.copy_(g_local)
model.segs[2].grad_ready_hook(arena.params[3], arena.params[4])
model.segs[1].grad_ready_hook(arena.params[1], arena.params[2])          # produced down to element 1000 <= 1200: flush now
q = 64 * world
assert 1000 <= red2._sent < 1000 + q, red2._sent          # nothing but the head (rounded to a shard boundary) is left for finish()
n_before = red2.launched
model.segs[0].grad_ready_hook(arena.params[0], arena.params[0])
red2.finish()
assert red2.launched == n_before + 1 and close(arena.grad, expect)
red2.paused = True
red2.start_step(); arena.grad.copy_(g_local)
model.segs[2].grad_ready_hook(arena.params[3], arena.params[4]); red2.finish()
assert red2.launched == 0 and torch.equal(arena.grad, g_local)
try:
    GradReducer(model, mode='ring')
    raise SystemExit('unknown mode accepted')
except ValueError:
    pass
dist.barrier(); dist.destroy_process_group()
print('OK', rank)
'''


@pytest.mark.parametrize('mode,wire,port', [('all_reduce', 'f32', 29541), ('rs_ag', 'f32', 29542), ('all_reduce', 'bf16', 29543), ('rs_ag', 'bf16', 29544)])
def test_grad_reducer_two_ranks_gloo(tmp_path, mode, wire, port):
    """Both exchange forms (one all-reduce per bucket | reduce-scatter + all-gather per bucket) and both wire dtypes really run
    with two ranks -- rs_ag no longer degrades to all_reduce on a non-RCCL backend -- plus the per-step accounting of stats()."""
    script = tmp_path / 'ddp_worker.py'
    script.write_text(DDP_WORKER)
    env = dict(os.environ, MASTER_ADDR='127.0.0.1', MASTER_PORT=str(port), WORLD_SIZE='2')
    procs = [subprocess.Popen([sys.executable, str(script), ROOT, mode, wire], env=dict(env, RANK=str(r)), stdout=subprocess.PIPE,
                              stderr=subprocess.STDOUT, text=True) for r in range(2)]
    outs = [p.communicate(timeout=240)[0] for p in procs]
    for p, o in zip(procs, outs):
        assert p.returncode == 0 and 'OK' in o, o


def test_grad_reducer_three_ranks_tail_bucket_not_divisible(tmp_path):
    """rs_ag on a world that does not divide the arena (3, 5, 6 or 7 ranks raised on every step):
    bucket edges are multiples of 64 * world, the tail bucket [0, first edge) of a 7801-element arena is 1081 elements = 1 mod 3
    and goes out as an all-reduce; the sum is the same."""
    script = tmp_path / 'ddp_worker.py'
    script.write_text(DDP_WORKER)
    env = dict(os.environ, MASTER_ADDR='127.0.0.1', MASTER_PORT='29547', WORLD_SIZE='3')
    procs = [subprocess.Popen([sys.executable, str(script), ROOT, 'rs_ag', 'f32', '1'], env=dict(env, RANK=str(r)), stdout=subprocess.PIPE,
                              stderr=subprocess.STDOUT, text=True) for r in range(3)]
    outs = [p.communicate(timeout=240)[0] for p in procs]
    for p, o in zip(procs, outs):
        assert p.returncode == 0 and 'OK' in o, o


def test_averaged_gradients_equal_single_process_gradients():
    """DDP equivalence on the oracle (CPU): mean of per-shard gradients == gradient of the concatenated batch when every
    loss is a mean over its elements (what the 1/world grad_scale of the fused optimizer relies on)."""
    from helpers import LOSS_WTS, build_oracle_model, oracle_step
    from oracle import avt_oracle as O
    orc = build_oracle_model('feat', 32, 64, 2, 4, 17)
    O.closed_form_fill_(list(orc.named_parameters()))
    g = torch.Generator().manual_seed(5)
    video = torch.rand((4, 6, 32, 1, 1, 1), generator=g); target = torch.randint(0, 17, (4,), generator=g)
    sub = torch.randint(-1, 17, (4, 6, 1), generator=g)
    oracle_step(orc, video, target, sub)
    full = {n: p.grad.clone() for n, p in orc.named_parameters()}
    acc = {n: torch.zeros_like(p) for n, p in orc.named_parameters()}
    for s in (slice(0, 2), slice(2, 4)):
        oracle_step(orc, video[s], target[s], sub[s])
        for n, p in orc.named_parameters():
            acc[n] += p.grad / 2
    for n in full:
        assert float((full[n] - acc[n]).abs().max()) <= 1e-5 * (1 + float(full[n].abs().max())), n


def test_bench_self_launch_refuses_more_ranks_than_devices():
    """`python bench.py --gpus N` spawns one rank per GPU itself; on a box with fewer devices it exits non-zero with a message
    (no silent single-GPU fallback).  Here: no GPU at all."""
    n = max(torch.cuda.device_count() + 1, 2)
    p = subprocess.run([sys.executable, os.path.join(ROOT, 'bench.py'), '--gpus', str(n), '--steps', '1', '--warmup', '0'],
                       capture_output=True, text=True, timeout=600)
    assert p.returncode != 0 and 'refusing to oversubscribe' in (p.stdout + p.stderr)


def test_fused_sgd_state_dict_is_torch_sgd_format():
    """Checkpoint interop (func/train.py:52-74, 760-769): the fused optimizer's state_dict has torch.optim.SGD's layout --
    structure checked here against a real torch.optim.SGD over same-shaped parameters (values are checked on the GPU)."""
    import inspect
    from avt_amd import optim
    src = inspect.getsource(optim.FusedSGD.state_dict)
    assert "'momentum_buffer'" in src and "'param_groups'" in src and "'state'" in src
    ps = [torch.nn.Parameter(torch.zeros(3, 2)), torch.nn.Parameter(torch.zeros(5))]
    ref = torch.optim.SGD([{'params': ps[:1]}, {'params': ps[1:], 'weight_decay': 0.1}], lr=0.1, momentum=0.9, nesterov=True)
    for p in ps:
        p.grad = torch.ones_like(p)
    ref.step()
    sd = ref.state_dict()
    assert set(sd) == {'state', 'param_groups'} and set(sd['state'][0]) == {'momentum_buffer'}
    assert {'lr', 'momentum', 'dampening', 'weight_decay', 'nesterov', 'params'} <= set(sd['param_groups'][0])


def test_init_model_partial_nonstrict_load(tmp_path):
    """func/train.py:457-497 semantics: container unwrapping, prefix filter + strip, shape-mismatch drop, unexpected keys ignored."""
    from helpers import build_oracle_model
    from avt_amd.func.train import init_from_model, init_model
    torch.manual_seed(0)
    src = build_oracle_model('vit', 128, 64, 2, 4, 17, vit=(128, 2, 2, 32))
    sd = {('module.' + k): v.clone() for k, v in src.state_dict().items()}
    sd['module.future_predictor.gpt_model.h.0.attn.bias'] = torch.ones(1, 1, 8, 8)           # HF 4.2.2 mask buffer
    sd['module.classifiers.action.weight'] = torch.zeros(99, 128)                             # another dataset's classifier
    path = tmp_path / 'ck.pth'
    torch.save({'model': sd, 'epoch': 3}, path)
    torch.manual_seed(1)
    dst = build_oracle_model('vit', 128, 64, 2, 4, 17, vit=(128, 2, 2, 32))
    keep_cls = dst.classifiers.action.weight.detach().clone()
    missing, unexpected = init_model(dst, str(path), 'module.')
    assert missing == ['classifiers.action.weight'] and unexpected == ['future_predictor.gpt_model.h.0.attn.bias']
    assert torch.equal(dst.classifiers.action.weight, keep_cls)
    for k, v in src.state_dict().items():
        if k != 'classifiers.action.weight':
            assert torch.equal(dst.state_dict()[k], v), k
    # the experiment-file form: [[backbone.model, <timm checkpoint>]] (expts/01_ek100_avt.txt:3) -- a bare state_dict
    torch.save(src.backbone.model.state_dict(), tmp_path / 'vit.pth')
    torch.manual_seed(2)
    dst2 = build_oracle_model('vit', 128, 64, 2, 4, 17, vit=(128, 2, 2, 32))
    init_from_model(dst2, [['backbone.model', str(tmp_path / 'vit.pth')]])
    for k, v in src.backbone.model.state_dict().items():
        assert torch.equal(dst2.backbone.model.state_dict()[k], v), k
    assert not torch.equal(dst2.future_predictor.encoder.weight, src.future_predictor.encoder.weight)


def test_gpu_clip_transform_draws_follow_the_reference_rules():
    """Host side of the GPU input pipeline: size / flip / crop draws (no GPU needed)."""
    import random
    from avt_amd.common.gpu_transforms import GpuClipTransform
    from oracle.avt_oracle import resize_shape
    random.seed(0); torch.manual_seed(0)
    tr = GpuClipTransform('248-280', -1, 224, train=True)
    seen_flip = set()
    for _ in range(50):
        nh, nw, flip, i, j = tr.draw(256, 456)
        assert 248 <= nh <= 280 and (nh, nw) == resize_shape(256, 456, nh) and 0 <= i <= nh - 224 and 0 <= j <= nw - 224
        seen_flip.add(flip)
    assert seen_flip == {0, 1}
    ev = GpuClipTransform(248, -1, 224, train=False)
    assert ev.draw(256, 456) == (248, 441, 0, 12, 108)          # centre crop: round((248-224)/2), round((441-224)/2)
    mc = GpuClipTransform(248, -1, 224, train=False, eval_num_crops=3, eval_flip_crops=True).eval_crops(256, 456)
    assert mc == [(248, 441, 0, 0, 0), (248, 441, 0, 12, 108), (248, 441, 0, 24, 217),
                  (248, 441, 1, 0, 217), (248, 441, 1, 12, 109), (248, 441, 1, 24, 0)]
    # ColorJitterVideo draws (torchvision 0.8.2 ColorJitter.get_params): a permutation of the active operations, factors in
    # [max(0, 1 - s), 1 + s] (hue: [-s, s]); inactive operations (strength 0) are left out; evaluation never jitters
    cj = GpuClipTransform(248, -1, 224, train=True, color_jitter_brightness=0.4, color_jitter_contrast=1.5, color_jitter_hue=0.1)
    orders = set()
    for _ in range(40):
        ops_ = cj.draw_jitter()
        assert sorted(o for o, _ in ops_) == [0, 1, 3]
        f = dict(ops_)
        assert 0.6 <= f[0] <= 1.4 and 0.0 <= f[1] <= 2.5 and -0.1 <= f[3] <= 0.1
        orders.add(tuple(o for o, _ in ops_))
    assert len(orders) > 2
    assert GpuClipTransform(248, -1, 224, train=True).draw_jitter() == []
    assert GpuClipTransform(248, -1, 224, train=False, color_jitter_hue=0.1).draw_jitter() == []
    with pytest.raises(ValueError):
        GpuClipTransform(248, -1, 224, train=True, color_jitter_hue=0.7)


def test_fragment_major_layout_queries_and_unpack():
    """ABI 7 on the host: avt_gemm_frag_ok / avt_gemm_frag_bytes answer without a GPU (the shape part of the persistent kernel's routing), and
    ops.gemm_frag_unpack is the inverse of the order csrc/gemm_persist.hip writes -- restated here element by element from the kernel's addressing
    (strip, column group, block, store, lane, value) -> (row, column)."""
    from avt_amd import ops, lib
    L = lib.load()
    assert L.avt_gemm_frag_ok(504320, 3072, 768) == 1 and L.avt_gemm_frag_ok(96 * 10 * 197, 4096, 1024) == 1      # config 2 / ViT-L at the bench's batches
    assert L.avt_gemm_frag_ok(3 * 10 * 197, 3072, 768) == 0          # 3 clips/GPU: too few tiles for the persistent kernel
    assert L.avt_gemm_frag_ok(504320, 3000, 768) == 0 and L.avt_gemm_frag_ok(504320, 3072, 8192) == 0 and L.avt_gemm_frag_ok(0, 3072, 768) == 0
    assert L.avt_gemm_frag_bytes(300, 128) == 384 * 128 * 2 and L.avt_gemm_frag_bytes(256, 64) == 256 * 64 * 2
    M, N = 300, 128
    ft = ops.FragTensor.__new__(ops.FragTensor)
    ft.M, ft.N = M, N
    S, C = (M + 127) // 128, N // 64
    buf = torch.full((S * C * 4 * 4 * 64 * 8,), -1.0)
    want = torch.zeros((S * 128, N))
    for s_ in range(S):
        for c in range(C):
            for i in range(4):
                for st in range(4):
                    for l in range(64):
                        for e in range(8):
                            j, q = st >> 1, 2 * (st & 1) + e // 4                      # pk_epi_gelu_block: store st = pieces (j, q0), (j, q0 + 1) of 4 values each
                            row = s_ * 128 + i * 32 + (l & 31)                         # accumulator layout: lane % 32 = row of the 32-row block
                            col = c * 64 + j * 32 + 8 * q + 4 * (l >> 5) + e % 4       # ... lane / 32 = which 4 of a piece's 8 columns
                            idx = ((((s_ * C + c) * 4 + i) * 4 + st) * 64 + l) * 8 + e
                            val = float(row * N + col)
                            buf[idx] = val; want[row, col] = val
    ft.buf = buf.to(torch.bfloat16).float()           # (values up to 49152 are not all bf16-exact: compare after the same rounding)
    got = ops.gemm_frag_unpack(ft)
    assert got.shape == (M, N) and torch.equal(got, want.to(torch.bfloat16).float()[:M])


def test_layernorm_fold_threshold():
    """HipViT folds LayerNorm into the qkv / fc1 GEMMs from fold_min_rows token rows on (measured crossover: 32 clips x 10 frames x 197 tokens; below it the
    unfolded path is faster, profiles/r05zh_fold_small_batch.txt); fold_layernorm = False switches it off everywhere, fold_min_rows = 0 on everywhere."""
    from avt_amd.models import vit
    class M: pass
    m = M(); m.fold_layernorm = True; m.fold_min_rows = 60000          # the product's defaults, restated (the autouse fixture zeroes the class attribute in here)
    assert vit.HipViT.fold_layernorm is True and vit.HipViT.fold_min_rows == 0
    assert not vit.use_fold(m, 3 * 10 * 197, 768, 11) and not vit.use_fold(m, 24 * 10 * 197, 768, 11)
    assert vit.use_fold(m, 32 * 10 * 197, 768, 11) and vit.use_fold(m, 256 * 10 * 197, 768, 11) and vit.use_fold(m, 96 * 10 * 197, 1024, 23)
    assert not vit.use_fold(m, 256 * 10 * 197, 768, 0) and not vit.use_fold(m, 256 * 10 * 197, 4096, 11)
    m.fold_layernorm = False
    assert not vit.use_fold(m, 256 * 10 * 197, 768, 11)
    m.fold_layernorm, m.fold_min_rows = True, 0
    assert vit.use_fold(m, 20, 256, 2)
    import inspect
    assert 'fold_min_rows = 60000' in inspect.getsource(vit.HipViT)


def test_gemm_variant_names_mirror_the_library_routing():
    """ops.gemm_variant names the kernel a GEMM lands on (the bench's per-kernel rows): the persistent 8-phase kernel for the big k-major
    contractions with K <= 4096 and a covered epilogue (csrc/gemm_persist.hip: avt_gemm_persist), gemm_8p_kernel for longer reductions,
    uncovered epilogues and other layouts."""
    from avt_amd import ops
    M = 2560 * 197
    assert ops.gemm_variant(M, 2304, 768, True, True, ops.OUT_BF16, 0, True) == 'gemm_8pp_kernel'            # qkv forward
    assert ops.gemm_variant(M, 3072, 768, True, True, ops.OUT_BF16, 0, True) == 'gemm_8pp_kernel'            # fc1 forward / fc2 data gradient
    assert ops.gemm_variant(M, 768, 3072, True, True, ops.OUT_BF16, 0, True) == 'gemm_8pp_kernel'            # fc2 forward (round 5: every K <= 4096)
    assert ops.gemm_variant(M, 768, 8192, True, True, ops.OUT_BF16, 0, True).startswith('gemm_8p_kernel')    # K > 4096
    assert ops.gemm_variant(M, 768, 768, True, True, ops.OUT_BF16, 0, False).startswith('gemm_8p_kernel')    # epilogue not covered
    assert ops.gemm_variant(M, 768, 768, True, False, ops.OUT_BF16, 0, True).startswith('gemm_8p_kernel')    # B not k-major
    assert ops.gemm_variant(M, 776, 768, True, True, ops.OUT_BF16, 0, True).startswith('gemm_8p_kernel')     # N % 256 != 0
    assert ops.gemm_variant(3940, 768, 768, True, True, ops.OUT_BF16, 0, True) != 'gemm_8pp_kernel'          # too few tiles
    assert ops.gemm_variant(M, 2304, 768, True, True, ops.OUT_BF16, 808, True).startswith('gemm_8p_kernel')  # forced one-tile-per-workgroup
    # small token counts (late round 5, profiles/r05z_small_batch_gemm_sweep.txt): all-k-major outputs of 96 .. 199 tiles of 256 x 256 take the 8-phase kernel,
    # below that the 3-deep 64 x 64 ring when K <= 3072; long reductions and the other layouts keep 128 x 128 tiles
    assert ops.gemm_variant(8 * 1970, 768, 768, True, True, ops.OUT_BF16, 0, True).startswith('gemm_8p_kernel')       # 8 clips: 186 tiles
    assert ops.gemm_variant(3 * 1970, 768, 3072, True, True, ops.OUT_BF16, 0, True).startswith('gemm_kernel<64,64,2,2,64,3')   # 3 clips: 72 tiles
    assert ops.gemm_variant(2560, 2048, 8192, True, True, ops.OUT_BF16, 0, True).startswith('gemm_kernel<128,128')     # head, K = 8192
    assert ops.gemm_variant(2560, 2048, 8192, True, False, ops.OUT_BF16, 0, True).startswith('gemm_kernel<128,128')    # head forward: B stored [K][N]
    assert ops.gemm_variant(2560, 3072, 768, True, True, ops.OUT_BF16, 0, True).startswith('gemm_8p_kernel')           # CLS-only last block's fc1: 120 tiles
    # the epilogue kind is part of the persistent kernel's name (rocprof shows gemm_8pp_kernel<EPK>)
    ek = ops.persist_epilogue_kind
    assert ek(ops.OUT_BF16, ops.ACT_NONE, True, False, False, False, False) == 0
    assert ek(ops.OUT_BF16, ops.ACT_GELU_ERF, True, False, False, True, False) == 1
    assert ek(ops.OUT_BF16, ops.ACT_NONE, True, True, False, False, False) == 2
    assert ek(ops.OUT_BF16, ops.ACT_MUL_AUX, False, False, True, False, True) == 3
    assert ek(ops.OUT_F32, ops.ACT_NONE, True, False, False, False, False) is None
    assert ek(ops.OUT_BF16, ops.ACT_NONE, True, True, False, False, False, res_period=197) is None
    assert ops.gemm_variant(M, 3072, 768, True, True, ops.OUT_BF16, 0, 1) == 'gemm_8pp_kernel<1>'


def test_bench_gemm_family_filter_catches_every_large_tile_kernel_the_router_can_return():
    """bench.py aggregates roofline.dominant_kernel / gemm_family / worst_large_gemm_row over ops.LARGE_TILE_KERNELS (round 4: the
    persistent kernel's name was missing from the bench's own tuple and 56 launches per step fell out of the numbers).  Every name
    gemm_variant can produce for a tile of >= 128 rows -- automatic routing over the step's shapes and every forced tile -- must match,
    and the small-tile names must not."""
    import itertools
    import re
    from avt_amd import ops
    src = open(os.path.join(ROOT, 'bench.py')).read()
    assert 'BIG = ops.LARGE_TILE_KERNELS' in src and src.count('startswith(BIG)') >= 3
    big = ops.LARGE_TILE_KERNELS
    M = 2560 * 197
    shapes = [(M, 2304, 768), (M, 3072, 768), (M, 768, 3072), (M, 768, 768), (M, 768, 2304), (2304, 768, M), (3072, 768, M), (768, 3072, M),
              (768, 768, M), (2560, 2048, 8192), (2560, 8192, 2048), (2560, 6144, 2048), (2048, 8192, 2560), (2560, 3840, 2048), (96 * 197 * 10, 4096, 1024)]
    seen = set()
    for (m, n, k), ak, bk, mode, epk in itertools.product(shapes, (True, False), (True, False), (ops.OUT_BF16, ops.OUT_F32, ops.OUT_ACCUM_F32),
                                                         (None, 0, 1, 2, 3)):
        for tile in (0, 128, 256, 808, 809, 2568):
            name = ops.gemm_variant(m, n, k, ak, bk, mode, tile, epk)
            seen.add(name.split('<')[0])
            rows = re.match(r'gemm_kernel<(\d+),', name)
            if rows is None or int(rows.group(1)) >= 128:
                assert name.startswith(big), name
    assert {'gemm_8pp_kernel', 'gemm_8p_kernel', 'gemm_kernel'} <= seen
    for tile in (64, 643):
        assert not ops.gemm_variant(3940, 768, 768, True, True, ops.OUT_BF16, tile, None).startswith(big)


def test_indirect_seed_packing_and_capture_slots():
    """ABI 9 (include/avt_hip.h "captured steps"): an indirect seed = bit 63 | offset << 48 | device address of the base seed; `+` adds to the offset, the
    way the modules derive a layer's seeds from the forward's base seed; inside a capture every fresh() takes the next slot and draw() refills the slots
    from the generators, in order (here on CPU memory: the packing is address arithmetic)."""
    import itertools
    import torch
    from avt_amd import seeds
    d = seeds.DevSeed(0x7f12_3456_7890)
    s = d + 16 * 3 + 2
    v = int(s)
    assert v >> 63 == 1 and (v >> 48) & 0x7FFF == 50 and v & ((1 << 48) - 1) == 0x7f12_3456_7890 and int(d + 0) == (1 << 63) | 0x7f12_3456_7890
    assert int(2 + d) == int(d + 2)
    with pytest.raises(AssertionError):
        int(d + (1 << 15))
    c1, c2 = itertools.count(1), itertools.count(100)
    g1, g2 = (lambda: next(c1) * 1000003), (lambda: (next(c2) * 7) & 0x7FFFFFFFFFFFFFFF)
    assert seeds.fresh(g1) == 1000003                      # eager: the value itself
    cap = seeds.SeedCapture(torch.device('cpu'), max_slots=4)
    with seeds.capturing(cap):
        a, b = seeds.fresh(g1), seeds.fresh(g2)
        assert isinstance(a, seeds.DevSeed) and b.ptr == a.ptr + 8 and a.ptr == cap.dev.data_ptr()
    assert seeds._capture is None and seeds.fresh(g2) == 700 and next(c1) == 2          # recording drew nothing from g1
    cap.draw()
    assert cap.dev[:2].tolist() == [3 * 1000003, 101 * 7]
    cap.draw()
    assert cap.dev[:2].tolist() == [4 * 1000003, 102 * 7]


def test_skinny_routing_mirror():
    """ops.gemm_variant restates gemm_impl's round-6 routing: at most 64 rows of k-major A rows go to the skinny kernel."""
    from avt_amd import ops
    assert ops.gemm_variant(30, 2048, 8192, True, True, ops.OUT_BF16, 0) == 'gemm_skinny_kernel<1>'
    assert ops.gemm_variant(30, 2048, 8192, True, False, ops.OUT_BF16, 0) == 'gemm_skinny_kernel<0>'
    assert ops.gemm_variant(45, 2048, 8192, True, True, ops.OUT_BF16, 0) == 'gemm_skinny_kernel<1>'          # 3 clips x 15 frames
    assert ops.gemm_variant(45, 2048, 8192, True, False, ops.OUT_BF16, 0).startswith('gemm_kernel<64,64,2,2,64,3')   # ... B stored [K][N]: the 64 x 64 ring
    assert ops.gemm_variant(65, 2048, 8192, True, True, ops.OUT_BF16, 0).startswith('gemm_kernel<64,64,2,2,64,3')
    assert 'skinny' not in ops.gemm_variant(30, 2048, 8192, False, False, ops.OUT_ACCUM_F32, 0)                    # weight gradients: not this kernel


def test_zeroed_gradient_registry():
    """ops.mark_zeroed / _first_write (round 6): the first write into a region of a registered buffer is 'fresh', an overlapping later one is not, regions
    outside every registered buffer never are, and an entry dies with its tensor (a freed buffer's address may be handed to a tensor nobody zeroed)."""
    import gc
    import torch
    from avt_amd import ops
    ops.forget_zeroed()
    buf = torch.zeros(4096)
    a, b = buf[:1024].view(32, 32), buf[1024:2048].view(32, 32)
    assert not ops._first_write(a, 32)                      # nothing registered
    ops.mark_zeroed(buf)
    assert ops._first_write(a, 32) and not ops._first_write(a, 32)
    assert not ops._first_write(buf[512:1536].view(32, 32), 32)            # overlaps a
    assert not ops._first_write(b, 32)                                      # ... and that attempt counted as a write into half of b
    assert ops._first_write(buf[2048:3072].view(32, 32), 16) and not ops._first_write(buf[2048:3072].view(32, 32), 32)
    other = torch.zeros(1024).view(32, 32)
    assert not ops._first_write(other, 32)
    ops.mark_zeroed(buf)                                                    # the optimizer stepped: everything is fresh again
    assert ops._first_write(a, 32)
    n = len(ops._ZEROED)
    del buf, a, b
    gc.collect()
    assert len(ops._ZEROED) == n - 1


def test_zeroed_gradient_registry_against_a_brute_force_model():
    """The registry keeps the written intervals sorted and merged; against a byte map over 2000 random writes: 'fresh' exactly when no byte of the
    region was written before."""
    import random
    import torch
    from avt_amd import ops
    ops.forget_zeroed()
    buf = torch.zeros(4096)
    ops.mark_zeroed(buf)
    written = [False] * 4096
    rng = random.Random(5)
    base = buf.data_ptr()
    for _ in range(2000):
        if rng.random() < 0.02:
            ops.mark_zeroed(buf)
            written = [False] * 4096
        cols = rng.choice([1, 2, 4, 8, 16])
        rows = rng.randint(1, 8)
        ld = cols * rng.choice([1, 1, 2])
        start = rng.randint(0, 4096 - rows * ld)
        view = torch.as_strided(buf, (rows, cols), (ld, 1), start)
        lo, hi = start, start + (rows - 1) * ld + cols           # the region the kernel may touch: first to last element
        want = not any(written[lo:hi])
        assert ops._first_write(view, rows) == want
        for i in range(lo, hi):
            written[i] = True
    los, his = ops._ZEROED[base][1]
    assert los == sorted(los) and all(h <= l for h, l in zip(his[:-1], los[1:]))
    ops.forget_zeroed()


def test_bench_fractions_keep_four_digits_however_slow_the_step():
    """The executed part of a step is smaller than the whole also where both are below a thousandth of the peak."""
    import bench
    assert bench.four_digits(0.38424) == 0.3842 and bench.four_digits(0.000914351) == 0.0009144 and bench.four_digits(0.0) == 0.0
    whole, skipped = bench.flops_per_clip(768, 12, 10), bench.flops_skipped_per_clip(768, 10)
    for clips in (0.5, 2.5, 975.2):
        assert bench.four_digits(clips * (whole - skipped) / 1e12 / 2500) < bench.four_digits(clips * whole / 1e12 / 2500)
