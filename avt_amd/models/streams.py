"""Live clips of different lengths on one AVT-h: the serving counterpart of the head's roll-out (reference models/future_prediction.py:168-202, which takes a
batch of clips of ONE length through HF's ``past_key_values``).

A stream is a clip that is still being watched.  ``append`` takes each stream's new frames -- none, one or a chunk, another number for every stream -- and
returns what the head decodes behind each of them; ``rollout`` predicts on from every stream's newest frame and leaves the streams as they were; ``release``
frees a stream for another clip.  The attention rounds its probabilities to bf16 (ops.paged_attn), which the roll-out of a batch does not.  Keys and values of all layers live in pages of one pool (include/avt_hip.h, ABI 10), so memory goes to the frames that
were seen and not to the longest clip there could be, and a step costs what its tokens cost.  Forward only, no dropout.

    streams = model.future_predictor.open_streams(64)
    decoded = streams.append(feats, counts)      # feats (sum(counts), C): stream 0's new frames, stream 1's, ...
    future = streams.rollout(4)                  # (64, 4, C): what follows each stream's newest frame
"""
import torch

from .. import ops
from ..arena import get_arena


class HeadStreams:
    """``streams``: how many clips at once; ``max_len``: frames of the longest (at most, and by default, the head's n_positions); ``page``: tokens of a page (a
    power of two from 8 to 1024); ``pages``: pages of the pool (default: every stream at its longest); ``weight_bits`` 4: the blocks' four projections run on 4-bit
    weights with group scales (ops.W4Weight), made here from the weights as they are.  That is for steps of few tokens (6 layers of 2048: 64 streams, one frame each, at 500, 1.1 ms
    a step and 2.4 in 16 bits; 0.8 and 1.2 of these are the kernels'); chunks of hundreds of rows are slower than in 16 bits (16 x 192 frames: 10 ms and 3.8)."""

    def __init__(self, head, streams, max_len=None, page=16, pages=None, weight_bits=16):
        n_pos = head.gpt_model.wpe.weight.size(0)
        self.max_len = n_pos if max_len is None else int(max_len)
        if streams < 1 or not 1 <= self.max_len <= n_pos:
            raise ValueError(f'open_streams: at least one stream of 1 to {n_pos} frames (got {streams}, {max_len})')
        if page < 8 or page > 1024 or page & (page - 1):
            raise ValueError(f'open_streams: the page must be a power of two from 8 to 1024 (got {page})')
        if weight_bits not in (4, 16):
            raise ValueError(f'open_streams: weight_bits must be 16 or 4 (got {weight_bits})')
        self.head, self.S, self.page = head, int(streams), int(page)
        self.width = -(-self.max_len // self.page)
        self.pages = self.S * self.width if pages is None else int(pages)
        if self.pages < 1:
            raise ValueError('open_streams: at least one page')
        if self.S > 4096:
            raise ValueError(f'open_streams: at most 4096 streams (got {streams})')
        if self.pages * self.page > 1 << 31:
            raise ValueError(f'open_streams: a pool of at most 2^31 rows (got {self.pages} pages of {self.page})')
        if head.inter_dim // head.n_head > 1024:
            raise ValueError(f'open_streams: heads of at most 1024 columns (got {head.inter_dim // head.n_head})')
        dev = head.encoder.weight.device
        arena = get_arena(head)                                # (raises off the GPU: there is no CPU path)
        E, H = head.inter_dim, head.n_head
        i32 = dict(device=dev, dtype=torch.int32)
        self.lens, self.owned = torch.zeros(self.S, **i32), torch.zeros(self.S, **i32)
        self.table = torch.zeros((self.S, self.width), **i32)
        self.free, self.n_free = torch.arange(self.pages, **i32), torch.full((1,), self.pages, **i32)
        self.caches = [tuple(torch.empty((self.pages, self.page, H, E // H), device=dev, dtype=torch.bfloat16) for _ in range(2)) for _ in head.gpt_model.h]
        self.last = torch.zeros((self.S, E), device=dev, dtype=torch.bfloat16)      # hidden state behind each stream's newest frame
        # what the host knows of the same numbers, so that a step that cannot be served is refused before anything runs
        self._lens, self._owned, self._n_free = [0] * self.S, [0] * self.S, self.pages
        self._w4 = None
        if weight_bits == 4:
            arena.refresh_shadow()
            self._w4 = [{n: self._quantize(lin.weight) for n, lin in (('c_attn', b.attn.c_attn), ('c_proj', b.attn.c_proj), ('c_fc', b.mlp.c_fc), ('m_proj', b.mlp.c_proj))}
                        for b in head.gpt_model.h]

    @staticmethod
    def _quantize(weight):
        """HF Conv1D weight (in, out) -> 4-bit [out, in] with the widest groups that divide it."""
        k = weight.size(0)
        group = next((g for g in (128, 64, 32) if k % g == 0), None)
        if group is None:
            raise ValueError(f'open_streams: 4-bit weights need layer widths that are multiples of 32 (got {k})')
        return ops.W4Weight.quantize(weight.detach().t(), group)

    @property
    def lengths(self):
        """Frames seen by each stream."""
        return list(self._lens)

    def _take(self, lens, counts):
        """Would the pool serve these counts?  Refuses, or returns (owned pages afterwards, free pages afterwards)."""
        owned, free = list(self._owned), self._n_free
        for s, (l, c) in enumerate(zip(lens, counts)):
            if l + c > self.max_len:
                raise ValueError(f'stream {s}: {l} + {c} frames are more than its {self.max_len}')
            need = max(0, -(-(l + c) // self.page) - owned[s])
            owned[s] += need
            free -= need
        if free < 0:
            raise ValueError(f'{-free} pages short: release streams, or open more pages')
        return owned, free

    def _plan(self, lens, counts, owned, n_free):
        """A plan from (lens, owned, n_free) on the device, for counts that _take has let through.  It writes new entries into the table behind the owned ones and
        nothing else: the pages are taken when the caller keeps the plan's owned and n_free, and free as before if it does not."""
        new = torch.tensor(counts, dtype=torch.int32).to(self.lens.device)
        return ops.paged_plan(lens, new, owned, self.table, self.free, n_free, self.page, sum(counts))

    def _linear(self, layer, name, lin, x, **kw):
        if self._w4 is not None:
            return ops.w4_linear(x, self._w4[layer][name], bias=lin.bias, **kw)
        return ops.conv1d_fwd(x, get_arena(self.head).sh(lin.weight), bias=lin.bias, **kw)

    def _blocks(self, enc, plan, counts, host_lens):
        """Input embeddings (N, E) of the plan's tokens -> their last hidden states (N, E)."""
        m, g, N = self.head, self.head.gpt_model, enc.size(0)
        E, H = m.inter_dim, m.n_head
        hd = E // H
        longest, cached = max(counts), max(l + c for l, c in zip(host_lens, counts))
        h = ops.embed_pos_fwd(enc, g.wpe.weight.detach().index_select(0, plan.positions), 1, N, E, 0.0, 0)
        for i, (blk, (kc, vc)) in enumerate(zip(g.h, self.caches)):
            l1, _, _ = ops.layernorm_fwd(h, blk.ln_1.weight, blk.ln_1.bias, m.ln_eps, save_stats=False)
            qkv = self._linear(i, 'c_attn', blk.attn.c_attn, l1)
            q, k, v = (qkv[:, j * E:(j + 1) * E].view(N, H, hd) for j in range(3))
            ops.paged_kv_write(k, v, kc, vc, plan.slots)
            att = ops.paged_attn(q, kc, vc, self.table, plan.cu, plan.kv_lens, max_new=longest, max_kv=cached)
            h1 = self._linear(i, 'c_proj', blk.attn.c_proj, att, res=h)
            l2, _, _ = ops.layernorm_fwd(h1, blk.ln_2.weight, blk.ln_2.bias, m.ln_eps, save_stats=False)
            a = self._linear(i, 'c_fc', blk.mlp.c_fc, l2, act=ops.ACT_GELU_TANH)
            h = self._linear(i, 'm_proj', blk.mlp.c_proj, a, res=h1)
        return ops.layernorm_fwd(h, g.ln_f.weight, g.ln_f.bias, m.ln_eps, save_stats=False)[0]

    def _decode(self, hidden):
        return ops.linear_fwd(hidden, get_arena(self.head).sh(self.head.decoder.weight), out_mode=ops.OUT_F32)

    @torch.no_grad()
    def append(self, feats, counts):
        """feats (N, C): the new frames' features, stream 0's first; counts: how many each stream gets (sum N).  Returns the decoded features behind each (N, C) fp32."""
        counts = [int(c) for c in counts]
        if len(counts) != self.S or min(counts) < 0 or feats.dim() != 2 or feats.size(0) != sum(counts) or feats.size(1) != self.head.in_features:
            raise ValueError(f'append: ({sum(counts)}, {self.head.in_features}) features for {self.S} counts, got {tuple(feats.shape)} for {len(counts)}')
        if not any(counts):
            return feats.new_zeros((0, feats.size(1)), dtype=torch.float32)
        if feats.device != self.lens.device:
            raise ValueError(f'append: features on device {feats.device}, streams on {self.lens.device}')
        arena = get_arena(self.head)
        arena.refresh_shadow()
        owned, free = self._take(self._lens, counts)
        plan = self._plan(self.lens, counts, self.owned, self.n_free)
        enc = ops.linear_fwd(feats.to(torch.bfloat16).contiguous(), arena.sh(self.head.encoder.weight))
        hidden = self._blocks(enc, plan, counts, self._lens)
        who = [s for s, c in enumerate(counts) if c]
        ends = torch.tensor([sum(counts[:s + 1]) - 1 for s in who], device=feats.device)
        decoded, last = self._decode(hidden), hidden.index_select(0, ends)
        who = torch.tensor(who, device=feats.device)
        # (kept only now: an error on the way here leaves the streams as they were)
        self.last.index_copy_(0, who, last)
        self.lens.copy_(plan.kv_lens)
        self.owned.copy_(plan.owned)
        self.n_free.copy_(plan.n_free)
        self._lens, self._owned, self._n_free = [l + c for l, c in zip(self._lens, counts)], owned, free
        return decoded

    @torch.no_grad()
    def rollout(self, steps):
        """(S, steps, C) fp32: entry 0 is decoded from the hidden state behind each stream's newest frame, entry i from the state reached by feeding the states back
        i times.  The streams keep their frames only, and the pool has its pages back afterwards (it has to hold those of the steps while they run); streams without
        frames give zeros."""
        if steps < 1:
            raise ValueError('rollout: at least one step')
        arena = get_arena(self.head)
        arena.refresh_shadow()
        live = [s for s, l in enumerate(self._lens) if l]
        out = self.last.new_zeros((self.S, steps, self.head.in_features), dtype=torch.float32)
        if not live:
            return out
        rows = torch.tensor(live, device=self.last.device)
        counts = [int(l > 0) for l in self._lens]
        self._take(self._lens, [c * (steps - 1) for c in counts])      # (all steps, or none)
        hidden, host = self.last.index_select(0, rows), list(self._lens)
        lens, owned, n_free = self.lens, self.owned, self.n_free       # (followed from step to step and not kept: the pages are the pool's again afterwards)
        for i in range(steps):
            out[rows, i] = self._decode(hidden)
            if i + 1 < steps:
                plan = self._plan(lens, counts, owned, n_free)
                hidden = self._blocks(hidden, plan, counts, host)
                lens, owned, n_free, host = plan.kv_lens, plan.owned, plan.n_free, [l + c for l, c in zip(host, counts)]
        return out

    def release(self, which):
        """Streams ``which`` give their pages back and are empty."""
        which = {int(s) for s in which}
        if any(not 0 <= s < self.S for s in which):
            raise ValueError(f'release: streams 0 to {self.S - 1}, got {sorted(which)}')
        for s in which:
            n = self._owned[s]
            self.free[self._n_free:self._n_free + n].copy_(self.table[s, :n])
            self._n_free += n
            self._lens[s] = self._owned[s] = 0
            self.lens[s] = 0
            self.owned[s] = 0
        self.n_free.fill_(self._n_free)
