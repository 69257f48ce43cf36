"""golem's Qwen3 dense decoder (qwen/) with every step on the device.

qwen.Model.ForwardBatch (qwen/model.go:127-175) for M consecutive positions:
the embedding rows (TokenEmbd.Row, a Q6_K dequantisation), then per block
(qwen/block.go:32-102):

    gx_norm_quant      x += previous FFN output; RMSNormPlain(attn_norm); Q8_0
    gx_qwen_qkv_rope   Q, K and V, stacked by rows into one Q4_0 matrix, then
                       head norms, RoPE, fp16 query, fp16 cache entries (for
                       a batch in the product's epilogue: gx_matmul_q4_0 +
                       gx_qwen_qk_rope bit for bit)
    gx_qwen_attention  scores, softmax, values; Q8_0 of the heads
    gx_matmul_q4_0     O
    gx_norm_quant      x += attention; RMSNormPlain(ffn_norm); Q8_0
    gx_matmul_q4_0     Gate and Up, stacked with rows interleaved by 32
    gx_swiglu_quant    silu(gate) * up; Q8_0
    gx_matmul_q4_0     Down

and the final norm (the last block's residual folded in).  Logits
(qwen/model.go:181-194) is QuantizeK plus the tied Q6_K head; greedy picks the
largest logit, the lower id on ties.  Stacking Q/K/V and Gate/Up changes no
result: every output row is its own product.

One position (a decode step) takes fewer launches: each pre-norm runs inside
the product after it (gx_norm_matmul_q4_0 for Q|K|V), and the FFN's norm,
Gate|Up product, SwiGLU and Q8_0 are one kernel (gx_norm_swiglu_q4_0), and
the head norms, RoPE, cache store and attention are one kernel
(gx_qwen_rope_attention), the same values bit for bit.

Every kernel treats a position on its own, so a prompt read in one batch
gives, bit for bit, what the same tokens give one at a time (golem's
TestBatchAgreesWithOneAtATime, qwen/model_test.go:79).

A decode step (one position) can be captured once into a HIP graph and
replayed: the token and its position are read from the device (the previous
step's argmax and a device counter), and the attention is launched for the
whole cache (max_pos = context - 1; the kernels stop at each position's own
prefix), so every replay runs the same launches.  A replay computes exactly
what the eager step computes.

Drafted tokens run as trees, one a conversation, in one pass
(forward_tree): gx_qwen_tree_plan, then the blocks with gx_qwen_qkv_rope
storing into draft buffers and gx_qwen_attention_tree reading the caches and
those.  verify_tree (gx_tree_verify) walks each tree by the target's logits and
commit_tree (gx_qwen_cache_commit) puts the kept path into the caches;
speculate is the loop over the three.

Pages (set_pages) hold conversations beside the slots: as many as there are
pages for, of any length up to the context, common beginnings once.
forward_pages reads new tokens of several of them in one pass, pages_step decodes
a batch in lock step: the blocks with gx_qwen_qk_rope_paged and
gx_qwen_attention_paged.  set_rope_scaling stretches the rotations of every
kind of pass to longer contexts (gx_rope_tables).
"""
import contextlib
import ctypes
import math
import weakref

import numpy as np
import torch

from . import capi

# gx_qwen_rope_attention reads at most this many cached positions (the
# one-kernel decode attention's limit); longer prefixes take the two calls.
FUSED_ATTENTION_MAX = 767


def rope_tables(dims, context, base):
    """RoPETable.Prepare (nn/rope.go:33-59) for positions 0 .. context-1:
    theta = pos * base^(-2i/dims) in float64, cos and sin rounded to float32,
    through the C library's pow, cos and sin."""
    half = dims // 2
    cos = np.empty((context, half), np.float32)
    sin = np.empty((context, half), np.float32)
    freqs = [math.pow(base, -2 * float(i) / float(dims)) for i in range(half)]
    for p in range(context):
        for i in range(half):
            theta = float(p) * freqs[i]
            cos[p, i] = math.cos(theta)
            sin[p, i] = math.sin(theta)
    return cos, sin


def interleave_rows(gate, up, rows, cols):
    """Gate and Up (Q4_0, rows x cols each) stacked into one matrix with
    their rows interleaved by 32: 32 gate rows, the same 32 up rows, and so
    on.  A 64-row tile then holds both halves of 32 SwiGLU outputs."""
    rb = cols // 32 * 18
    g = np.asarray(gate, np.uint8).reshape(rows // 32, 32 * rb)
    u = np.asarray(up, np.uint8).reshape(rows // 32, 32 * rb)
    return np.ascontiguousarray(np.concatenate([g, u], axis=1)).reshape(-1)


class _Q8:
    """A Q8_0 batch on the device: q [M][K], scales and qsum [M][K/32]."""

    def __init__(self, M, K):
        self.q = torch.empty((M, K), dtype=torch.int8, device="cuda")
        self.s = torch.empty((M, K // 32), dtype=torch.float32, device="cuda")
        self.qs = torch.empty((M, K // 32), dtype=torch.int32, device="cuda")


class _Step(torch.cuda.CUDAGraph):
    """A model's captured step.  Every replay puts its own tokens and hidden
    states in the place of those of a pass over drafted tokens."""

    model = None  # a weak reference's proxy: the model holds its steps

    def replay(self):
        self.model.tree_states = False
        self.model.page_batch = None
        super().replay()


class QwenModel:
    """attention: "parallel" runs decode steps' attention with its softmax
    total and value sums in a parallel order (gx_qwen_rope_attention_parallel
    / gx_qwen_attention_parallel) and prompts (more than four positions) on
    the matrix cores: golem's values within float rounding, so a prompt read
    in one batch and the same tokens read one at a time agree only to that
    rounding.  "golem" keeps golem's serial order bit for bit, and with it
    golem's batch == one at a time.  Trees of drafted tokens (forward_tree) run
    in one order under both, another than either's."""

    def __init__(self, ctx, cfg, weights, max_batch, attention="parallel"):
        if attention not in ("parallel", "golem"):
            raise ValueError(f"qwen: attention order {attention!r}")
        self.ctx, self.cfg, self.max_batch = ctx, cfg, max_batch
        self.graph = None
        self.slot_graphs = {}  # captured lock-step slot steps, by conversation count
        self.set_attention(attention)
        vp, call = capi.vp, capi.call
        qd, kvd = cfg.heads * cfg.head_dim, cfg.kv_heads * cfg.head_dim
        self.qd, self.kvd = qd, kvd

        def dev(a, dtype=torch.float32):
            return torch.from_numpy(np.ascontiguousarray(a)).to(dtype).cuda()

        self.blocks = []
        for b in weights["blocks"]:
            self.blocks.append({
                "qkv": capi.Weight(ctx, np.concatenate([b["q"], b["k"], b["v"]]), capi.Q4_0, qd + 2 * kvd, cfg.dim),
                "o": capi.Weight(ctx, b["o"], capi.Q4_0, cfg.dim, qd),
                "gu": capi.Weight(ctx, interleave_rows(b["gate"], b["up"], cfg.ffn, cfg.dim), capi.Q4_0,
                                  2 * cfg.ffn, cfg.dim),
                "down": capi.Weight(ctx, b["down"], capi.Q4_0, cfg.dim, cfg.ffn),
                "attn_norm": dev(b["attn_norm"]), "ffn_norm": dev(b["ffn_norm"]),
                "q_norm": dev(b["q_norm"]), "k_norm": dev(b["k_norm"]),
            })
        # the tied embedding / head: Q6_K (config 3) or Q4_0 (a pure Q4_0 checkpoint)
        self.head_quant = weights.get("token_embd_quant", capi.Q6_K)
        if self.head_quant not in (capi.Q6_K, capi.Q4_0):
            raise ValueError("qwen: the tied head must be Q6_K or Q4_0")
        self.embd = capi.Weight(ctx, weights["token_embd"], self.head_quant, cfg.vocab, cfg.dim)
        self.output_norm = dev(weights["output_norm"])
        # a row for every position of the cache (a multiple of 8), as the
        # kernels' contract has it
        cos, sin = rope_tables(cfg.head_dim, (cfg.max_context + 7) // 8 * 8, cfg.rope_base)
        self.rope_cos, self.rope_sin = dev(cos), dev(sin)
        # one conversation until set_slots says otherwise
        self._make_caches(1)

        M = max_batch
        self.xs = torch.empty((M, cfg.dim), dtype=torch.float32, device="cuda")
        self.xs2 = torch.empty((1, cfg.dim), dtype=torch.float32, device="cuda")  # the fused steps' other residual
        self.x8 = _Q8(M, cfg.dim)
        self.qkv = torch.empty((M, qd + 2 * kvd), dtype=torch.float32, device="cuda")
        self.qh = torch.empty((M, qd), dtype=torch.int16, device="cuda")
        self.set8 = _Q8(M, qd)
        self.attn = torch.empty((M, cfg.dim), dtype=torch.float32, device="cuda")
        self.gu = torch.empty((M, 2 * cfg.ffn), dtype=torch.float32, device="cuda")
        self.mid8 = _Q8(M, cfg.ffn)
        self.ffn = torch.empty((M, cfg.dim), dtype=torch.float32, device="cuda")
        self.hidden = torch.empty((M, cfg.dim), dtype=torch.float32, device="cuda")
        self.positions = torch.empty((M,), dtype=torch.int32, device="cuda")
        self.slot_ids = torch.zeros((M,), dtype=torch.int32, device="cuda")  # each token's conversation
        self.tokens = torch.empty((M,), dtype=torch.int32, device="cuda")
        self.k8 = torch.empty((M, cfg.dim), dtype=torch.int8, device="cuda")
        self.ks = torch.empty((M, cfg.dim // 256), dtype=torch.float32, device="cuda")
        self.bs = torch.empty((M, cfg.dim // 16), dtype=torch.int16, device="cuda")
        self.logit = torch.empty((M, cfg.vocab), dtype=torch.float32, device="cuda")
        self.next_id = torch.empty((M,), dtype=torch.int32, device="cuda")
        self.pos_dev = torch.zeros((1,), dtype=torch.int32, device="cuda")  # the graph's position counter
        self.history = torch.zeros((cfg.max_context + 1,), dtype=torch.int32, device="cuda")
        self.graph = None
        self.slot_graphs = {}
        self.drafts = 0  # tokens the draft buffers hold (set_drafts)
        self.tree_ws, self.tree_ws_kept = None, []
        self.pool, self.conversations = None, 0  # pages (set_pages), and the conversations opened in any so far
        self.page_batch, self.page_graphs = None, {}  # the conversations in lock step, their captured steps
        self.page_ws = None
        self.tree_states = False  # the tokens and hidden states are forward_tree's
        n = capi.size_out("gx_qwen_attention_workspace_bytes", M, cfg.heads, cfg.max_context - 1)
        self.attn_ws = torch.empty((n + 255) // 256 * 256, dtype=torch.uint8, device="cuda")
        self._vp, self._call = vp, call

    def _make_caches(self, n):
        """n conversations of max_context // n positions each (SetSlots,
        qwen/slots.go:19-37).  Per layer, keys in 16-byte pieces
        [slot][kv_head][head_dim/8][context][8] and values transposed
        [slot][kv_head][head_dim][context]."""
        cfg = self.cfg
        self.nslots, self.slot = n, 0
        self.slot_context = cfg.max_context // n
        self.context = (self.slot_context + 7) // 8 * 8
        kshape = (n, cfg.kv_heads, cfg.head_dim // 8, self.context, 8)
        vshape = (n, cfg.kv_heads, cfg.head_dim, self.context)
        self.kc = self.vc = None
        self.kc = [torch.zeros(kshape, dtype=torch.int16, device="cuda") for _ in range(cfg.layers)]
        self.vc = [torch.zeros(vshape, dtype=torch.int16, device="cuda") for _ in range(cfg.layers)]
        self.tree = None  # a pass over drafted tokens read the caches being replaced

    def set_attention(self, attention):
        """Switch the decode steps' attention order ("parallel" or "golem");
        a captured step is dropped."""
        if attention not in ("parallel", "golem"):
            raise ValueError(f"qwen: attention order {attention!r}")
        sfx = "_parallel" if attention == "parallel" else ""
        self._rope_attention, self._attention = "gx_qwen_rope_attention" + sfx, "gx_qwen_attention" + sfx
        self.graph = None
        self.slot_graphs = {}

    def set_slots(self, n):
        """SetSlots (qwen/slots.go:19-37): n independent conversations, each
        holding max_context // n positions; replaces whatever was cached."""
        if n < 1:
            raise ValueError(f"qwen: {n} slots")
        if self.cfg.max_context // n < 1:
            raise ValueError(f"qwen: a context of {self.cfg.max_context} cut into {n} slots leaves no position each")
        self.graph = None  # a captured step addressed the caches being replaced
        self.slot_graphs = {}
        self._make_caches(n)

    def use_slot(self, i):
        """UseSlot (qwen/slots.go:62-78): forward() goes to conversation i."""
        if not 0 <= i < self.nslots:
            raise IndexError(f"qwen: slot {i} of {self.nslots}")
        self.slot = i

    def reset(self):
        """Forget the conversations (Model.Reset): the caches are cleared."""
        for k, v in zip(self.kc, self.vc):
            k.zero_()
            v.zero_()

    def _mm(self, w, act, M, y, ldy):
        vp = self._vp
        self._call("gx_matmul_q4_0", self.ctx.ptr, w.ptr, vp(act.q), vp(act.s), vp(act.qs), None, M, 0, w.rows,
                   None, vp(y), ldy)

    def forward(self, tokens, start_pos):
        """ForwardBatch: tokens is a device int32 tensor of M ids (or a host
        sequence, uploaded); returns the device hidden states [M][dim] after
        the final norm (a view of reused storage)."""
        cfg = self.cfg
        if not torch.is_tensor(tokens):
            tokens = torch.tensor(np.asarray(tokens, dtype=np.int32), device="cuda")
        M = int(tokens.shape[0])
        if M > self.max_batch or start_pos + M > self.slot_context:
            raise ValueError(f"qwen: {M} positions from {start_pos} exceed the batch {self.max_batch} "
                             f"or the context {self.slot_context}")
        self.tokens[:M].copy_(tokens)
        torch.arange(start_pos, start_pos + M, dtype=torch.int32, out=self.positions[:M])
        if self.nslots > 1:
            self.slot_ids[:M].fill_(self.slot)
        self._blocks(M, start_pos + M - 1, own_slot=True)
        return self.hidden[:M]

    def forward_slots(self, tokens, slots, positions):
        """ForwardSlots (qwen/place.go:33-41): token i at position
        positions[i] of conversation slots[i], all in one pass over the
        weights; each token's arithmetic is what it would be alone.  Returns
        the device hidden states [M][dim] after the final norm."""
        M = len(tokens)
        if not (len(slots) == len(positions) == M) or M > self.max_batch or M == 0:
            raise ValueError(f"qwen: {M} tokens, {len(slots)} slots, {len(positions)} positions "
                             f"(batch {self.max_batch})")
        for sl, pos in zip(slots, positions):
            if not 0 <= sl < self.nslots:
                raise IndexError(f"qwen: slot {sl} of {self.nslots}")
            if not 0 <= pos < self.slot_context:
                raise ValueError(f"qwen: position {pos} is past a slot's {self.slot_context}")
        self.tokens[:M].copy_(torch.tensor(np.asarray(tokens, dtype=np.int32)))
        self.positions[:M].copy_(torch.tensor(np.asarray(positions, dtype=np.int32)))
        self.slot_ids[:M].copy_(torch.tensor(np.asarray(slots, dtype=np.int32)))
        self._blocks(M, int(max(positions)))
        return self.hidden[:M]

    def residual(self, tokens, start_pos, blocks):
        """The residual stream of M >= 2 consecutive tokens after the first
        `blocks` blocks (0: the embedding rows), as ForwardBatch computes it
        before the final norm: a host [M][dim] float32 copy.  For checking a
        deep model block by block."""
        M = len(tokens)
        if M < 2 or M > self.max_batch or start_pos + M > self.slot_context:
            raise ValueError(f"qwen: {M} positions from {start_pos} for a block-by-block residual")
        self.tokens[:M].copy_(torch.tensor(np.asarray(tokens, dtype=np.int32)))
        torch.arange(start_pos, start_pos + M, dtype=torch.int32, out=self.positions[:M])
        if self.nslots > 1:
            self.slot_ids[:M].fill_(self.slot)
        self._blocks(M, start_pos + M - 1, blocks, own_slot=True)
        self.ctx.sync()
        if blocks == 0:
            return self.xs[:M].cpu().numpy().copy()
        return (self.xs[:M] + self.ffn[:M]).cpu().numpy()  # the last block's residual add

    def _blocks(self, M, max_pos, blocks=None, one_per_slot=False, own_slot=False, attend=None):
        """The embedding rows, every block and the final norm for the M tokens
        and positions already in self.tokens / self.positions (with `blocks`:
        only the first that many blocks, and no final norm).  one_per_slot:
        the M tokens belong to M different conversations (a lock-step step),
        so the head norms, RoPE, cache stores and attention run as one
        kernel.  own_slot: the M tokens are the current conversation's
        (forward), whose caches the attention then reads as a lone
        conversation's.  attend(i): block i's head norms, RoPE, stores and
        attention from self.qkv to self.set8, in place of the caches'."""
        cfg, vp, call, ctx = self.cfg, self._vp, self._call, self.ctx.ptr
        self.tree_states = False
        self.page_batch = None
        call("gx_weight_rows", ctx, self.embd.ptr, 0, vp(self.tokens), M, vp(self.xs))
        if M == 1:
            return self._blocks_one(max_pos, attend)
        qd, kvd = self.qd, self.kvd
        sl = vp(self.slot_ids) if self.nslots > 1 else None
        for i, b in enumerate(self.blocks):
            if blocks is not None and i >= blocks:
                return
            add = None if i == 0 else vp(self.ffn)
            call("gx_norm_quant", ctx, vp(self.xs), cfg.dim, add, cfg.dim, vp(b["attn_norm"]), M, cfg.dim,
                 np.float32(cfg.eps), None, 0, vp(self.x8.q), vp(self.x8.s), vp(self.x8.qs))
            if attend is not None:
                self._mm(b["qkv"], self.x8, M, self.qkv, qd + 2 * kvd)
                attend(i)
            elif one_per_slot and max_pos < FUSED_ATTENTION_MAX:
                self._mm(b["qkv"], self.x8, M, self.qkv, qd + 2 * kvd)
                call("gx_qwen_rope_attention_slots", ctx, vp(self.qkv), qd + 2 * kvd, M, cfg.heads, cfg.kv_heads,
                     cfg.head_dim, max_pos, vp(self.positions), vp(b["q_norm"]), vp(b["k_norm"]),
                     vp(self.rope_cos), vp(self.rope_sin), np.float32(cfg.eps), vp(self.kc[i]), vp(self.vc[i]),
                     self.context, vp(self.set8.q), vp(self.set8.s), vp(self.set8.qs), sl, self.nslots,
                     1 if self._attention.endswith("_parallel") else 0)
            else:
                # the product and the heads' norms, RoPE and stores (one
                # kernel for a batch: the product's epilogue)
                call("gx_qwen_qkv_rope", ctx, b["qkv"].ptr, vp(self.x8.q), vp(self.x8.s), vp(self.x8.qs), M,
                     cfg.heads, cfg.kv_heads, cfg.head_dim, vp(self.positions), vp(b["q_norm"]), vp(b["k_norm"]),
                     vp(self.rope_cos), vp(self.rope_sin), np.float32(cfg.eps), vp(self.qh), vp(self.kc[i]),
                     vp(self.vc[i]), self.context, sl, self.nslots, vp(self.qkv))
                if sl is None or not own_slot:
                    kca, vca, sla = self.kc[i], self.vc[i], sl
                else:
                    # a prompt of the current conversation reads that slot's
                    # caches as a lone conversation's: the same kernels, and
                    # so the same values, as the model without slots
                    kca, vca, sla = self.kc[i][self.slot], self.vc[i][self.slot], None
                call(self._attention, ctx, vp(self.qh), M, cfg.heads, cfg.kv_heads, cfg.head_dim,
                     max_pos, vp(self.positions), vp(kca), vp(vca), self.context,
                     vp(self.set8.q), vp(self.set8.s), vp(self.set8.qs), vp(self.attn_ws), self.attn_ws.numel(),
                     sla, self.nslots if sla is not None else 0)
            self._mm(b["o"], self.set8, M, self.attn, cfg.dim)
            call("gx_norm_quant", ctx, vp(self.xs), cfg.dim, vp(self.attn), cfg.dim, vp(b["ffn_norm"]), M, cfg.dim,
                 np.float32(cfg.eps), None, 0, vp(self.x8.q), vp(self.x8.s), vp(self.x8.qs))
            # the product and SwiGLU + Q8_0 in one kernel (its epilogue)
            call("gx_matmul_swiglu_q4_0", ctx, b["gu"].ptr, vp(self.x8.q), vp(self.x8.s), vp(self.x8.qs), M,
                 vp(self.mid8.q), vp(self.mid8.s), vp(self.mid8.qs))
            self._mm(b["down"], self.mid8, M, self.ffn, cfg.dim)
        if blocks is not None:
            return
        call("gx_norm_quant", ctx, vp(self.xs), cfg.dim, vp(self.ffn), cfg.dim, vp(self.output_norm), M, cfg.dim,
             np.float32(cfg.eps), vp(self.hidden), cfg.dim, None, None, None)

    def _blocks_one(self, max_pos, attend=None):
        """The blocks for one position, with each pre-norm fused into the
        product after it, and the SwiGLU with its Q8_0 into the Gate/Up
        product (the same values bit for bit).  The residual moves between two buffers, since a
        fused product's workgroups all read it while one writes x + add."""
        cfg, vp, call, ctx = self.cfg, self._vp, self._call, self.ctx.ptr
        qd, kvd = self.qd, self.kvd
        sl = vp(self.slot_ids) if self.nslots > 1 else None
        eps = np.float32(cfg.eps)
        cur, other = self.xs, self.xs2
        for i, b in enumerate(self.blocks):
            if i == 0:
                call("gx_norm_matmul_q4_0", ctx, b["qkv"].ptr, vp(cur), None, vp(b["attn_norm"]), eps, None, 0,
                     b["qkv"].rows, vp(self.qkv))
            else:
                call("gx_norm_matmul_q4_0", ctx, b["qkv"].ptr, vp(cur), vp(self.ffn), vp(b["attn_norm"]), eps,
                     vp(other), 0, b["qkv"].rows, vp(self.qkv))
                cur, other = other, cur
            if attend is not None:
                attend(i)
            elif max_pos < FUSED_ATTENTION_MAX:  # head norms + RoPE + cache store + attention, one kernel
                call(self._rope_attention, ctx, vp(self.qkv), qd + 2 * kvd, cfg.heads, cfg.kv_heads,
                     cfg.head_dim, max_pos, vp(self.positions), vp(b["q_norm"]), vp(b["k_norm"]),
                     vp(self.rope_cos), vp(self.rope_sin), eps, vp(self.kc[i]), vp(self.vc[i]), self.context,
                     vp(self.set8.q), vp(self.set8.s), vp(self.set8.qs), sl, self.nslots)
            else:
                call("gx_qwen_qk_rope", ctx, vp(self.qkv), qd + 2 * kvd, 1, cfg.heads, cfg.kv_heads,
                     cfg.head_dim, vp(self.positions), vp(b["q_norm"]), vp(b["k_norm"]), vp(self.rope_cos),
                     vp(self.rope_sin), eps, vp(self.qh), vp(self.kc[i]), vp(self.vc[i]), self.context, sl,
                     self.nslots)
                call(self._attention, ctx, vp(self.qh), 1, cfg.heads, cfg.kv_heads, cfg.head_dim,
                     max_pos, vp(self.positions), vp(self.kc[i]), vp(self.vc[i]), self.context,
                     vp(self.set8.q), vp(self.set8.s), vp(self.set8.qs), vp(self.attn_ws), self.attn_ws.numel(),
                     sl, self.nslots)
            self._mm(b["o"], self.set8, 1, self.attn, cfg.dim)
            call("gx_norm_swiglu_q4_0", ctx, b["gu"].ptr, vp(cur), vp(self.attn), vp(b["ffn_norm"]), eps,
                 vp(other), vp(self.mid8.q), vp(self.mid8.s), vp(self.mid8.qs))
            cur, other = other, cur
            self._mm(b["down"], self.mid8, 1, self.ffn, cfg.dim)
        call("gx_norm_quant", ctx, vp(cur), cfg.dim, vp(self.ffn), cfg.dim, vp(self.output_norm), 1, cfg.dim,
             eps, vp(self.hidden), cfg.dim, None, None, None)

    def _decode_step(self):
        """One greedy step read entirely from the device: token self.tokens[0]
        at position self.pos_dev.  Leaves the next token in self.tokens[0] and
        in self.history[position + 1], and advances the position."""
        self._blocks(1, self.slot_context - 1)
        self.logits(0)
        # the argmax, straight into the next step's token, and the history
        # entry, counter and position of the next step, in one launch pair
        self._call("gx_argmax_step", self.ctx.ptr, self._vp(self.logit), self.cfg.vocab, self._vp(self.tokens),
                   self._vp(self.history), self.history.numel(), self._vp(self.pos_dev), self._vp(self.positions))

    def _capture(self, step):
        """step recorded into a graph.  The library's stream is the capture stream
        while recording, and then the context's own again."""
        torch.cuda.synchronize()
        stream, graph = torch.cuda.Stream(), _Step()
        graph.model = weakref.proxy(self)
        self._call("gx_set_stream", self.ctx.ptr, ctypes.c_void_p(stream.cuda_stream))
        try:
            with torch.cuda.graph(graph, stream=stream):
                step()
        finally:
            self._call("gx_set_stream", self.ctx.ptr, ctypes.c_void_p(self.ctx.stream))
        torch.cuda.synchronize()
        return graph

    def capture_decode(self):
        """Records _decode_step into a HIP graph (once)."""
        if self.graph is not None:
            return
        if self.nslots > 1:
            raise ValueError("qwen: the captured decode step serves one conversation")
        self.graph = self._capture(self._decode_step)

    def logits(self, row):
        """Logits of hidden state `row` (of the last forward): the tied head
        (qwen/model.go:181-194), Q6_K over the Q8_K form or Q4_0 over the Q8_0
        form; the device logits [vocab] (reused storage)."""
        cfg, vp, call, ctx = self.cfg, self._vp, self._call, self.ctx.ptr
        h = self.hidden[row:row + 1]
        if self.head_quant == capi.Q4_0:
            a = self.x8  # free once the blocks are done
            call("gx_quantize_q8_0", ctx, vp(h), cfg.dim, 1, cfg.dim, vp(a.q), vp(a.s), vp(a.qs), None, None)
            call("gx_matmul_q4_0", ctx, self.embd.ptr, vp(a.q), vp(a.s), vp(a.qs), None, 1, 0, cfg.vocab, None,
                 vp(self.logit), cfg.vocab)
            return self.logit[0]
        call("gx_quantize_q8_k", ctx, vp(h), cfg.dim, 1, cfg.dim, vp(self.k8), vp(self.ks), vp(self.bs))
        call("gx_matmul_q6_k", ctx, self.embd.ptr, vp(self.k8), vp(self.ks), vp(self.bs), 1, 0, cfg.vocab, None,
             vp(self.logit), cfg.vocab)
        return self.logit[0]

    def start_slots(self, tokens, positions):
        """Seeds lock-step decoding of conversations 0 .. n-1: token i (a
        host id, or a device int32 tensor of n ids) at position positions[i]
        of slot i."""
        n = len(positions)
        if not 0 < n <= min(self.nslots, self.max_batch):
            raise ValueError(f"qwen: {n} conversations for {self.nslots} slots")
        if max(positions) >= self.slot_context:
            raise ValueError(f"qwen: position {max(positions)} is past a slot's {self.slot_context}")
        t = tokens if torch.is_tensor(tokens) else torch.tensor(np.asarray(tokens, dtype=np.int32))
        self.tree_states, self.page_batch = False, None  # their tokens are replaced
        self.tokens[:n].copy_(t)
        self.positions[:n].copy_(torch.tensor(np.asarray(positions, dtype=np.int32)))
        if self.nslots > 1:
            self.slot_ids[:n].copy_(torch.arange(n, dtype=torch.int32))
        self._slot_pos = list(positions)

    def slots_step(self, n, graph=False):
        """One lock-step decode step of conversations 0 .. n-1 from the
        tokens and positions on the device (the server's batch of slots,
        cmd/golem-server/runner.go:233-297): one pass over the weights and one
        head read for all n; the next ids replace the tokens (and stay in
        next_id[:n]) and every position advances.  graph: the step as a
        replay of its captured form (capture_slots), the same values bit for
        bit."""
        top = max(self._slot_pos)
        if top >= self.slot_context:
            raise ValueError(f"qwen: position {top} is past a slot's {self.slot_context}")
        if graph:
            self.capture_slots(n)
            self.slot_graphs[n].replay()
        else:
            self._slots_device_step(n, top)
        self._slot_pos = [p + 1 for p in self._slot_pos]
        return self.next_id[:n]

    def _slots_device_step(self, n, max_pos):
        self._blocks(n, max_pos, one_per_slot=self.nslots > 1)
        self.logits_batch(range(n))
        # the picks, each row's next token and its position advanced, in one launch
        self._call("gx_argmax_slots_step", self.ctx.ptr, self._vp(self.logit), self.cfg.vocab, n, self.cfg.vocab,
                   self._vp(self.next_id), self._vp(self.tokens), self._vp(self.positions))

    def capture_slots(self, n):
        """Records the device work of slots_step(n) into a HIP graph (once per
        n): the attention is launched for a slot's whole context and each
        token stops at its own prefix, read from the device, so one recording
        serves every step."""
        if self.slot_graphs.get(n) is not None:
            return
        if not 0 < n <= min(self.nslots, self.max_batch):
            raise ValueError(f"qwen: {n} conversations for {self.nslots} slots")
        self.slot_graphs[n] = self._capture(lambda: self._slots_device_step(n, self.slot_context - 1))

    def logits_batch(self, rows):
        """LogitsBatch (qwen/model.go:200-214): the logits of several hidden
        states of the last forward in one read of the head; device [n][vocab]
        (reused storage), each row what logits() gives it alone."""
        cfg, vp, call, ctx = self.cfg, self._vp, self._call, self.ctx.ptr
        rows = list(rows)
        n = len(rows)
        if not 0 < n <= self.max_batch:
            raise ValueError(f"qwen: {n} states for a batch of {self.max_batch}")
        if rows == list(range(rows[0], rows[0] + n)):
            h = self.hidden[rows[0]:rows[0] + n]
        else:
            h = self.attn[:n]  # free once the blocks are done
            h.copy_(self.hidden[rows])
        if self.head_quant == capi.Q4_0:
            a = self.x8
            call("gx_quantize_q8_0", ctx, vp(h), cfg.dim, n, cfg.dim, vp(a.q), vp(a.s), vp(a.qs), None, None)
            call("gx_matmul_q4_0", ctx, self.embd.ptr, vp(a.q), vp(a.s), vp(a.qs), None, n, 0, cfg.vocab, None,
                 vp(self.logit), cfg.vocab)
        else:
            call("gx_quantize_q8_k", ctx, vp(h), cfg.dim, n, cfg.dim, vp(self.k8), vp(self.ks), vp(self.bs))
            call("gx_matmul_q6_k", ctx, self.embd.ptr, vp(self.k8), vp(self.ks), vp(self.bs), n, 0, cfg.vocab, None,
                 vp(self.logit), cfg.vocab)
        return self.logit[:n]

    def next_tokens(self, rows):
        """The greedy ids after several hidden states (one head read), left
        on the device: next_id[:n]."""
        n = len(list(rows))
        self.logits_batch(rows)
        self._call("gx_argmax", self.ctx.ptr, self._vp(self.logit), self.cfg.vocab, n, self.cfg.vocab,
                   self._vp(self.next_id))
        return self.next_id[:n]

    def next_token(self, row):
        """The greedy id after hidden state `row`, left on the device."""
        self.logits(row)
        self._call("gx_argmax", self.ctx.ptr, self._vp(self.logit), self.cfg.vocab, 1, self.cfg.vocab,
                   self._vp(self.next_id))
        return self.next_id[:1]

    def greedy(self, prompt, steps, graph=False):
        """The prompt in one batch, then `steps` greedy tokens, each fed back
        from the device (graph: the decode steps as replays of the captured
        step).  Returns the ids (host list)."""
        if len(prompt) + steps - 1 > self.cfg.max_context:
            raise ValueError(f"qwen: {steps} tokens after {len(prompt)} exceed the context {self.cfg.max_context}")
        self.reset()
        self.forward(prompt, 0)
        tok = self.next_token(len(prompt) - 1)
        if graph:
            self.capture_decode()
            self.start_decode(tok, len(prompt))
            for _ in range(steps - 1):
                self.graph.replay()
            return self.decoded(len(prompt), steps)
        ids = []
        pos = len(prompt)
        for s in range(steps):
            ids.append(tok.clone())
            if s + 1 < steps:
                self.forward(tok, pos)
                tok = self.next_token(0)
                pos += 1
        return [int(t.item()) for t in ids]

    def start_decode(self, tok, pos):
        """Seeds the captured step: token `tok` (device) at position `pos`,
        also recorded as the history's entry `pos`."""
        if pos >= self.cfg.max_context:
            raise ValueError(f"qwen: position {pos} is past the context {self.cfg.max_context}")
        self.tree_states, self.page_batch = False, None  # their tokens are replaced
        self.tokens[:1].copy_(tok)
        self.history[pos:pos + 1].copy_(tok)
        self.pos_dev.fill_(pos)
        self.positions[:1].fill_(pos)

    def decoded(self, pos, steps):
        """The ids of `steps` greedy tokens from position `pos`: the seed
        and those the replays left in the history."""
        return [int(t) for t in self.history[pos:pos + steps].cpu().tolist()]

    # ---- drafted tokens ----

    def set_drafts(self, tokens):
        """Draft buffers for passes of up to `tokens` drafted tokens, roots
        included (at most max_batch): a layer's keys and values in the caches'
        layouts, a token a row."""
        cfg, dev = self.cfg, "cuda"
        if not 0 < tokens <= self.max_batch:
            raise ValueError(f"qwen: {tokens} drafted tokens for a batch of {self.max_batch}")
        self.drafts, self.tree = tokens, None
        self.draft_context = (tokens + 7) // 8 * 8
        kshape = (cfg.kv_heads, cfg.head_dim // 8, self.draft_context, 8)
        vshape = (cfg.kv_heads, cfg.head_dim, self.draft_context)
        self.kd = [torch.zeros(kshape, dtype=torch.int16, device=dev) for _ in range(cfg.layers)]
        self.vd = [torch.zeros(vshape, dtype=torch.int16, device=dev) for _ in range(cfg.layers)]
        half = cfg.head_dim // 2
        self.draft_cos = torch.empty((tokens, half), dtype=torch.float32, device=dev)
        self.draft_sin = torch.empty((tokens, half), dtype=torch.float32, device=dev)
        self.draft_rows = torch.empty((tokens,), dtype=torch.int32, device=dev)

    def _tree_workspace(self, name, *size):
        n = (capi.size_out(name, *size) + 255) // 256 * 256
        if self.tree_ws is None or self.tree_ws.numel() < n:
            self.tree_ws_kept.append(self.tree_ws)  # a captured pass may hold its address
            self.tree_ws = torch.empty(n, dtype=torch.uint8, device="cuda")
        return self._vp(self.tree_ws), self.tree_ws.numel()

    def forward_tree(self, tokens, parents, prefixes, slots=None):
        """One pass over a tree of drafted tokens for each of several
        conversations.  tokens[b] and parents[b] list tree b's nodes: node 0
        is the token decided on and not yet run (parent -1), every other
        node's parent an earlier one.  prefixes[b] counts the positions
        conversation slots[b] (default: the current slot, for one tree) has
        cached.  Returns the device hidden states [M][dim] after the final
        norm, the trees' nodes one after another; the caches stay as they are
        until commit_tree.  The attention's sums are in an order of their own:
        a node's state is what its path run alone gives but for float rounding
        (and what that moves in the Q8_0 activations after it).  A token outside
        the vocabulary may be among the drafts (verify_tree passes it over),
        but its NaN entries make every layer's attention sum the rest of its
        tree again key by key, many times the pass without it.  As any pass
        does, this one replaces the device's tokens and positions: seed a
        lock-step or captured decode again after it."""
        n, sizes = len(tokens), [len(t) for t in tokens]
        slots = [self.slot] * n if slots is None else list(slots)
        M, nodes = sum(sizes), max(sizes, default=0)
        if not len(parents) == len(prefixes) == len(slots) == n or n == 0 or min(sizes) == 0:
            raise ValueError("qwen: a tree needs tokens, parents, a prefix and a slot")
        if M > self.drafts:
            raise ValueError(f"qwen: {M} drafted tokens for buffers of {self.drafts} (set_drafts)")
        if len(set(slots)) != n:
            raise ValueError("qwen: two trees of one conversation")
        for t, p, prefix, slot in zip(tokens, parents, prefixes, slots):
            if not 0 <= slot < self.nslots:
                raise IndexError(f"qwen: slot {slot} of {self.nslots}")
            depth = []
            for i, up in enumerate(p):
                if len(p) != len(t) or not (up == -1 if i == 0 else 0 <= up < i):
                    raise ValueError(f"qwen: node {i}'s parent {up} is no earlier node")
                depth.append(0 if i == 0 else depth[up] + 1)
            if prefix < 0 or prefix + max(depth) >= self.slot_context:
                raise ValueError(f"qwen: position {prefix + max(depth)} is past the context {self.slot_context}")

        def dev(v):
            return torch.tensor(np.asarray(v, dtype=np.int32), device="cuda")

        def flat(v):
            return [x for row in v for x in row]

        first = np.concatenate([[0], np.cumsum(sizes)])
        ids = dev(flat(tokens))
        tree = {"n": n, "M": M, "nodes": nodes, "first": dev(first), "parents": dev(flat(parents)),
                "prefix": dev(prefixes), "slots": dev(slots), "max_prefix": int(max(prefixes)),
                "mask": torch.empty((M, (nodes + 31) // 32), dtype=torch.int32, device="cuda"),
                "path": torch.full((n, nodes), -1, dtype=torch.int32, device="cuda"),
                "counts": torch.zeros((n,), dtype=torch.int32, device="cuda"),
                "next": torch.empty((n,), dtype=torch.int32, device="cuda")}
        self.tree = None  # none to judge until this one is whole
        self.tokens[:M].copy_(ids)
        self._tree_blocks(tree)
        self.tree = tree
        return self.hidden[:M]

    def _tree_blocks(self, t):
        """The embedding rows, blocks and final norm of forward_tree, from the
        device state alone (so that it can be captured, the workspace being
        there)."""
        cfg, vp, call, ctx = self.cfg, self._vp, self._call, self.ctx.ptr
        n, M, nodes = t["n"], t["M"], t["nodes"]
        eps = np.float32(cfg.eps)
        self.tree_states, self.page_batch = False, None
        call("gx_qwen_tree_plan", ctx, n, M, nodes, vp(t["first"]), vp(t["parents"]), vp(t["prefix"]),
             vp(self.rope_cos), vp(self.rope_sin), cfg.head_dim // 2, self.slot_context, vp(self.draft_rows),
             vp(self.positions), vp(t["mask"]), vp(self.draft_cos), vp(self.draft_sin))
        call("gx_weight_rows", ctx, self.embd.ptr, 0, vp(self.tokens), M, vp(self.xs))
        ws, size = self._tree_workspace("gx_qwen_attention_tree_workspace_bytes", n, M, nodes, cfg.heads,
                                        cfg.kv_heads, cfg.head_dim, t["max_prefix"])
        for i, b in enumerate(self.blocks):
            call("gx_norm_quant", ctx, vp(self.xs), cfg.dim, None if i == 0 else vp(self.ffn), cfg.dim,
                 vp(b["attn_norm"]), M, cfg.dim, eps, None, 0, vp(self.x8.q), vp(self.x8.s), vp(self.x8.qs))
            # the drafts' own buffers as caches, the plan's rows as positions
            call("gx_qwen_qkv_rope", ctx, b["qkv"].ptr, vp(self.x8.q), vp(self.x8.s), vp(self.x8.qs), M,
                 cfg.heads, cfg.kv_heads, cfg.head_dim, vp(self.draft_rows), vp(b["q_norm"]), vp(b["k_norm"]),
                 vp(self.draft_cos), vp(self.draft_sin), eps, vp(self.qh), vp(self.kd[i]), vp(self.vd[i]),
                 self.draft_context, None, 0, vp(self.qkv))
            call("gx_qwen_attention_tree", ctx, vp(self.qh), n, M, nodes, vp(t["first"]), vp(t["mask"]),
                 vp(t["prefix"]), t["max_prefix"], cfg.heads, cfg.kv_heads, cfg.head_dim, vp(self.kc[i]),
                 vp(self.vc[i]), self.context, vp(self.kd[i]), vp(self.vd[i]), self.draft_context, None,
                 vp(self.set8.q), vp(self.set8.s), vp(self.set8.qs), ws, size, vp(t["slots"]), self.nslots)
            self._mm(b["o"], self.set8, M, self.attn, cfg.dim)
            call("gx_norm_quant", ctx, vp(self.xs), cfg.dim, vp(self.attn), cfg.dim, vp(b["ffn_norm"]), M, cfg.dim,
                 eps, None, 0, vp(self.x8.q), vp(self.x8.s), vp(self.x8.qs))
            call("gx_matmul_swiglu_q4_0", ctx, b["gu"].ptr, vp(self.x8.q), vp(self.x8.s), vp(self.x8.qs), M,
                 vp(self.mid8.q), vp(self.mid8.s), vp(self.mid8.qs))
            self._mm(b["down"], self.mid8, M, self.ffn, cfg.dim)
        call("gx_norm_quant", ctx, vp(self.xs), cfg.dim, vp(self.ffn), cfg.dim, vp(self.output_norm), M, cfg.dim,
             eps, vp(self.hidden), cfg.dim, None, None, None)
        self.tree_states = True

    def verify_tree(self, temperature=0.0, draft_logits=None, draft_temperature=None, uniforms=None):
        """The walk down the trees of the last forward_tree by the target's
        logits (gx_tree_verify): temperature 0 keeps the drafts that greedy
        decoding would have drawn; above, each node's number in `uniforms`
        (device float32 [M], in [0, 1); default: torch's generator) decides,
        the drafts being given tokens or, with draft_logits (device [M][vocab],
        the draft model's logits after each node), drawn from the softmax of
        their parent's row at draft_temperature (default: temperature),
        siblings without replacement in their order: only then are the tokens
        distributed as the target's own.  No other pass may have run
        since: the model's own are noticed and refused, replays of a graph that
        a caller captured over them are not.  Returns device tensors:
        path [trees][nodes] (-1 behind), counts [trees], next [trees]."""
        t, vp, V = self._a_tree(), self._vp, self.cfg.vocab
        M = t["M"]
        if not self.tree_states:
            raise ValueError("qwen: another pass has replaced the drafted tokens' states")
        if uniforms is None and temperature > 0:
            uniforms = torch.rand((M,), device="cuda")
        for x, shape, what in ((draft_logits, (M, V), "draft logits"), (uniforms, (M,), "random numbers")):
            if x is not None and not (tuple(x.shape) == shape and x.dtype == torch.float32
                                      and x.device == self.tokens.device and x.is_contiguous()):
                raise ValueError(f"qwen: the {what} are a contiguous float32 {shape} on {self.tokens.device}, not "
                                 f"{x.dtype} {tuple(x.shape)} on {x.device}")
        logits = self.logits_batch(range(M))
        ws, size = self._tree_workspace("gx_tree_verify_workspace_bytes", t["n"], M, V)
        self._call("gx_tree_verify", self.ctx.ptr, vp(logits), V, t["n"], M, t["nodes"], V, vp(t["first"]),
                   vp(t["parents"]), vp(self.tokens), vp(draft_logits), V, temperature,
                   temperature if draft_temperature is None else draft_temperature, vp(uniforms), vp(t["path"]),
                   vp(t["counts"]), vp(t["next"]), ws, size)
        return t["path"], t["counts"], t["next"]

    def commit_tree(self):
        """The kept paths of the last verify_tree (none before it) into their
        conversations' caches: prefixes[b] + counts[b] positions are cached
        then."""
        t, vp, cfg = self._a_tree(), self._vp, self.cfg
        layers = [(ctypes.c_void_p * cfg.layers)(*[x.data_ptr() for x in xs])
                  for xs in (self.kc, self.vc, self.kd, self.vd)]
        self._call("gx_qwen_cache_commit", self.ctx.ptr, cfg.layers, *layers, t["n"], t["M"], t["nodes"],
                   vp(t["first"]), vp(t["path"]), vp(t["counts"]), vp(t["prefix"]), cfg.kv_heads, cfg.head_dim,
                   self.context, self.draft_context, vp(t["slots"]), self.nslots)

    def _a_tree(self):
        if self.tree is None:
            raise ValueError("qwen: no pass over drafted tokens (forward_tree)")
        return self.tree

    def fork_slot(self, src, dsts, length):
        """The first `length` positions of conversation src into each of dsts:
        conversations with a common beginning read it once."""
        cfg, dsts = self.cfg, list(dsts)
        if not 0 <= length <= self.slot_context:
            raise ValueError(f"qwen: {length} positions of a slot's {self.slot_context}")
        layers = [(ctypes.c_void_p * cfg.layers)(*[x.data_ptr() for x in xs]) for xs in (self.kc, self.vc)]
        self._call("gx_qwen_cache_fork", self.ctx.ptr, cfg.layers, *layers, self.nslots, cfg.kv_heads, cfg.head_dim,
                   self.context, src, (ctypes.c_int32 * len(dsts))(*dsts), len(dsts), length)

    def speculate(self, prompt, steps, draft, temperature=0.0, generator=None):
        """`steps` tokens after the prompt, several a pass where drafts are
        kept.  draft(ids) proposes a tree after the ids so far: (tokens,
        parents) of nodes 1, 2, .., parents as node numbers with 0 the last
        id, or with a third entry (or None), the device draft logits
        [1 + nodes][vocab] that the tokens were drawn from: each node's from its
        parent's row at `temperature`, siblings without replacement
        (verify_tree).  temperature 0: the target's best tokens, which are
        greedy()'s unless two logits are closer than the orders of the
        attention's sums move them (forward_tree); above, random numbers come
        from `generator` (a torch generator of the GPU).  Returns the ids and
        the number of passes."""
        if not prompt or len(prompt) + steps - 1 > self.slot_context:
            raise ValueError(f"qwen: {steps} tokens after {len(prompt)} exceed the context {self.slot_context}")
        if self.drafts == 0:
            self.set_drafts(self.max_batch)
        ids, passes, cached = [int(x) for x in prompt], 0, len(prompt) - 1
        for at in range(0, cached, self.max_batch):
            self.forward(ids[at:min(cached, at + self.max_batch)], at)
        while len(ids) < len(prompt) + steps:
            tokens, parents, *logits = draft(list(ids))
            depth, keep = [0], 1  # nodes within the context and the buffers
            for p in parents[:self.drafts - 1]:
                depth.append(depth[p] + 1)
                if cached + depth[-1] >= self.slot_context:
                    break
                keep += 1
            tree = [ids[-1]] + [int(x) for x in tokens[:keep - 1]]
            self.forward_tree([tree], [[-1] + list(parents[:keep - 1])], [cached])
            uniforms = None if temperature == 0 else torch.rand((keep,), generator=generator, device="cuda")
            path, counts, nxt = self.verify_tree(temperature, logits[0][:keep] if logits and logits[0] is not None else None,
                                                 uniforms=uniforms)
            self.commit_tree()
            count, after = int(counts[0]), int(nxt[0])
            if after < 0:
                raise ValueError("qwen: logits that no token can be drawn from")
            kept = path[0, :count].tolist()
            ids += [tree[i] for i in kept[1:]] + [after]
            cached += count
            passes += 1
        return ids[len(prompt):len(prompt) + steps], passes

    # ---- rotations of long contexts ----

    def set_rope_scaling(self, kind, factor=1.0, original=None, low=1.0, high=None, magnitude=None):
        """The rotations of every pass from now on: "plain" (as the model was
        built), "linear" (positions divided by factor), "ramp" or "turns"
        (gx_rope_tables: pairs that turn more than `high` times in the
        `original` context stay, those that turn less than `low` times are
        divided; high is 32 for "ramp", 4 for "turns").  magnitude multiplies
        cosines and sines: 0.1 ln(factor) + 1 for "ramp", else 1.  What is
        cached already keeps the rotation it was stored with: reset, or start
        conversations anew."""
        cfg = self.cfg
        kinds = {"plain": capi.ROPE_PLAIN, "linear": capi.ROPE_LINEAR, "ramp": capi.ROPE_RAMP, "turns": capi.ROPE_TURNS}
        if kind not in kinds:
            raise ValueError(f"qwen: a rotation scaled by {kind!r}")
        if kind in ("ramp", "turns") and original is None:
            raise ValueError("qwen: the original context is missing")
        if kind == "plain":
            cos, sin = rope_tables(cfg.head_dim, self.rope_cos.shape[0], cfg.rope_base)
            self.rope_cos.copy_(torch.from_numpy(cos))
            self.rope_sin.copy_(torch.from_numpy(sin))
            return
        high = (32.0 if kind == "ramp" else 4.0) if high is None else high
        magnitude = (0.1 * math.log(factor) + 1.0 if kind == "ramp" else 1.0) if magnitude is None else magnitude
        self._call("gx_rope_tables", self.ctx.ptr, cfg.head_dim, cfg.rope_base, kinds[kind], factor, original or 0, low,
                   high, magnitude, 0, self.rope_cos.shape[0], self._vp(self.rope_cos), self._vp(self.rope_sin))

    # ---- pages ----

    def set_pages(self, count, size=64, kind="fp16"):
        """A pool of `count` pages of `size` positions (a power of two from 16
        to 1024) a layer, for conversations beside the slots'; replaces the
        last pool and its conversations, whose numbers are not given out again.
        kind: "fp16", or "int8" with a scale for each head and position, in
        half the bytes."""
        cfg, dev = self.cfg, "cuda"
        if count < 1 or size < 16 or size > 1024 or size & (size - 1):
            raise ValueError(f"qwen: {count} pages of {size} positions (a power of two from 16 to 1024)")
        if kind not in ("fp16", "int8"):
            raise ValueError(f"qwen: pages of {kind!r}")
        if cfg.head_dim not in (32, 64, 96, 128):
            raise ValueError(f"qwen: pages hold heads of 32, 64, 96 and 128, not {cfg.head_dim}")
        shape = (count, cfg.kv_heads, size, cfg.head_dim)
        dtype = torch.int16 if kind == "fp16" else torch.int8
        # (what works on the last one first: a captured step holds its addresses)
        self.pool, self.page_batch, self.page_graphs, self.page_ws = None, None, {}, None
        self.pool = {
            "count": count, "size": size, "kind": capi.PAGES_F16 if kind == "fp16" else capi.PAGES_I8,
            "k": [torch.zeros(shape, dtype=dtype, device=dev) for _ in range(cfg.layers)],
            "v": [torch.zeros(shape, dtype=dtype, device=dev) for _ in range(cfg.layers)],
            "ks": [torch.zeros(shape[:3], device=dev) if kind == "int8" else None for _ in range(cfg.layers)],
            "vs": [torch.zeros(shape[:3], device=dev) if kind == "int8" else None for _ in range(cfg.layers)],
            "free": list(range(count - 1, -1, -1)), "held": [0] * count,  # pages, and how many conversations hold each
            "lists": {}, "lengths": {},                                   # conversations' pages and positions
        }

    def _a_pool(self):
        if self.pool is None:
            raise ValueError("qwen: no pages (set_pages)")
        return self.pool

    def _a_conversation(self, c):
        p = self._a_pool()
        if c not in p["lists"]:
            raise IndexError(f"qwen: no conversation {c} in the pages")
        return p

    def open_conversation(self):
        """A conversation of no positions in the pages; its number."""
        p = self._a_pool()
        c = self.conversations
        self.conversations += 1
        p["lists"][c], p["lengths"][c] = [], 0
        return c

    def close_conversation(self, c):
        """Its pages go back to the pool, but for those another one shares."""
        p = self._a_conversation(c)
        for page in p["lists"].pop(c):
            p["held"][page] -= 1
            if p["held"][page] == 0:
                p["free"].append(page)
        del p["lengths"][c]
        if self.page_batch and c in self.page_batch:
            self.page_batch = None

    def share_conversation(self, c, length):
        """A new conversation whose first `length` positions, whole pages of
        them, are conversation c's own pages: nothing is copied."""
        p = self._a_conversation(c)
        if length % p["size"] or not 0 <= length <= p["lengths"][c]:
            raise ValueError(f"qwen: {length} of {p['lengths'][c]} positions are no whole pages of {p['size']}")
        new = self.open_conversation()
        p["lists"][new] = p["lists"][c][:length // p["size"]]
        for page in p["lists"][new]:
            p["held"][page] += 1
        p["lengths"][new] = length
        return new

    def conversation_length(self, c):
        return self._a_conversation(c)["lengths"][c]

    @contextlib.contextmanager
    def _grown(self, wanted):
        """A pass for which conversations c hold pages for wanted[c] positions: all
        of them, or none and an error.  Those taken for a pass that fails go back."""
        p = self.pool
        need = {c: (w + p["size"] - 1) // p["size"] - len(p["lists"][c]) for c, w in wanted.items()}
        if sum(max(x, 0) for x in need.values()) > len(p["free"]):
            raise ValueError(f"qwen: {sum(max(x, 0) for x in need.values())} pages wanted, {len(p['free'])} free")
        for c, x in need.items():
            for _ in range(x):
                page = p["free"].pop()
                p["held"][page] = 1
                p["lists"][c].append(page)
        try:
            yield
        except BaseException:
            for c, x in reversed(need.items()):
                for _ in range(x):
                    page = p["lists"][c].pop()
                    p["held"][page] = 0
                    p["free"].append(page)
            raise

    def _page_lists(self, conversations, width):
        table = np.full((len(conversations), width), -1, np.int32)
        for b, c in enumerate(conversations):
            pages = self.pool["lists"][c]
            table[b, :len(pages)] = pages
        return torch.from_numpy(table)

    def _attend_pages(self, i, t):
        """Block i's heads of a pass over pages: self.qkv into the pages, and their
        attention into self.set8."""
        cfg, vp, call, ctx, p = self.cfg, self._vp, self._call, self.ctx.ptr, self.pool
        eps, b = np.float32(cfg.eps), self.blocks[i]
        pool = (p["kind"], vp(p["k"][i]), vp(p["v"][i]), vp(p["ks"][i]), vp(p["vs"][i]), p["count"], p["size"],
                vp(t["table"]), t["table"].shape[1])
        call("gx_qwen_qk_rope_paged", ctx, vp(self.qkv), self.qd + 2 * self.kvd, t["M"], cfg.heads, cfg.kv_heads,
             cfg.head_dim, vp(self.positions), vp(t["owners"]), vp(b["q_norm"]), vp(b["k_norm"]), vp(self.rope_cos),
             vp(self.rope_sin), self.rope_cos.shape[0], cfg.head_dim, 0, eps, vp(self.qh), *pool, t["n"])
        call("gx_qwen_attention_paged", ctx, vp(self.qh), t["n"], t["M"], t["tokens"], vp(t["first"]), vp(t["lengths"]),
             t["bound"], cfg.heads, cfg.kv_heads, cfg.head_dim, *pool, None, vp(self.set8.q), vp(self.set8.s),
             vp(self.set8.qs), vp(self.page_ws), self.page_ws.numel())

    def _page_workspace(self, t):
        """A workspace for t's attention: the passes share one, which goes back to
        the allocator when a larger one takes its place (in stream order, as the
        pass's other tensors do), but for captured steps that hold it.  It at least
        doubles, so that what those hold is less than the one in use."""
        n = max(256, (capi.size_out("gx_qwen_attention_paged_workspace_bytes", t["n"], t["M"], t["tokens"], self.cfg.heads,
                                    self.cfg.kv_heads, self.cfg.head_dim, t["bound"]) + 255) // 256 * 256)
        if self.page_ws is None or self.page_ws.numel() < n:
            last = 0 if self.page_ws is None else self.page_ws.numel()
            self.page_ws = None
            self.page_ws = torch.empty(max(n, 2 * last), dtype=torch.uint8, device="cuda")

    def forward_pages(self, tokens, conversations):
        """One pass over new tokens of several conversations in the pages:
        tokens[b], at least one, follow what conversations[b] holds.  Returns the
        device hidden states [M][dim] after the final norm, the conversations'
        tokens one after another.  The attention's sums are in an order that
        hangs on the batch: a state is what the tokens give alone but for float
        rounding (and what that moves in the Q8_0 activations after it).  As any
        pass does, this one replaces the device's tokens and positions: seed a
        lock-step or captured decode again after it."""
        p, n, sizes = self._a_pool(), len(tokens), [len(x) for x in tokens]
        M = sum(sizes)
        if n == 0 or len(conversations) != n or min(sizes) == 0 or M > self.max_batch:
            raise ValueError(f"qwen: {M} tokens of {n} conversations for a batch of {self.max_batch}")
        if len(set(conversations)) != n:
            raise ValueError("qwen: a conversation twice in one batch")
        lengths = {}
        for c, x in zip(conversations, sizes):
            lengths[c] = self._a_conversation(c)["lengths"][c] + x
            if lengths[c] > self.cfg.max_context:
                raise ValueError(f"qwen: {lengths[c]} positions exceed the context {self.cfg.max_context}")
        with self._grown(lengths):
            self._pages_pass(tokens, conversations, sizes, lengths)
        for c in conversations:
            p["lengths"][c] = lengths[c]
        return self.hidden[:M]

    def _pages_pass(self, tokens, conversations, sizes, lengths):
        """forward_pages once the conversations hold the pages for lengths[c] positions."""
        p, n, M = self.pool, len(tokens), sum(sizes)

        def dev(v):
            return torch.tensor(np.asarray(v, dtype=np.int32), device="cuda")

        t = {"n": n, "M": M, "tokens": max(sizes), "first": dev(np.concatenate([[0], np.cumsum(sizes)])),
             "lengths": dev([lengths[c] for c in conversations]), "owners": dev(np.repeat(np.arange(n), sizes)),
             "bound": max(lengths.values()),
             "table": self._page_lists(conversations, max(len(p["lists"][c]) for c in conversations)).cuda()}
        self._page_workspace(t)
        ids = dev([y for x in tokens for y in x])
        at = dev(np.concatenate([np.arange(lengths[c] - x, lengths[c]) for c, x in zip(conversations, sizes)]))
        self.tree_states, self.page_batch = False, None  # their tokens are replaced
        self.tokens[:M].copy_(ids)
        self.positions[:M].copy_(at)
        self._blocks(M, 0, attend=lambda i: self._attend_pages(i, t))

    def start_pages(self, tokens, conversations):
        """Seeds lock-step decoding of conversations in the pages: token i (a
        host id, or a device int32 tensor of ids) follows what conversations[i]
        holds."""
        n, p = len(conversations), self._a_pool()
        if not 0 < n <= self.max_batch or len(set(conversations)) != n:
            raise ValueError(f"qwen: {n} conversations in lock step for a batch of {self.max_batch}")
        lengths = [self._a_conversation(c)["lengths"][c] for c in conversations]
        t = tokens if torch.is_tensor(tokens) else torch.tensor(np.asarray(tokens, dtype=np.int32))
        if t.shape != (n,):
            raise ValueError(f"qwen: {n} conversations for tokens of shape {tuple(t.shape)}")
        self.tree_states, self.page_batch = False, None  # their tokens are replaced
        self.tokens[:n].copy_(t)
        self.positions[:n].copy_(torch.tensor(np.asarray(lengths, dtype=np.int32)))
        self.page_batch = list(conversations)

    def pages_step(self, graph=False):
        """One lock-step decode step of the conversations that start_pages named:
        the next ids replace the tokens (and stay in next_id[:n]), every
        position advances.  Any other pass or seeding in between replaces the
        tokens: the step is refused then.  graph: as a replay of the captured
        step of this many conversations, the same values bit for bit; one is
        captured for each power of two that the longest conversation's length
        stays under."""
        p = self._a_pool()
        if not self.page_batch:
            raise ValueError("qwen: no conversations in lock step (start_pages)")
        batch, cfg = self.page_batch, self.cfg
        n, top = len(batch), 1 + max(p["lengths"][c] for c in batch)
        if top > cfg.max_context:
            raise ValueError(f"qwen: {top} positions exceed the context {cfg.max_context}")
        with self._grown({c: p["lengths"][c] + 1 for c in batch}):
            self._pages_one_step(n, min(cfg.max_context, max(256, 1 << (top - 1).bit_length())), graph)
        for c in batch:
            p["lengths"][c] += 1
        self.page_batch = batch
        return self.next_id[:n]

    def _pages_one_step(self, n, bound, graph):
        """pages_step once the conversations hold the pages for one position more, for
        lengths of at most `bound`."""
        p, batch = self.pool, self.page_batch
        if (n, bound) not in self.page_graphs:
            width = (bound + p["size"] - 1) // p["size"]
            t = {"n": n, "M": n, "tokens": 1, "bound": bound, "first": torch.arange(n + 1, dtype=torch.int32, device="cuda"),
                 "lengths": torch.empty((n,), dtype=torch.int32, device="cuda"),
                 "owners": torch.arange(n, dtype=torch.int32, device="cuda"),
                 "table": torch.empty((n, width), dtype=torch.int32, device="cuda"), "graph": None}
            self.page_graphs[n, bound] = t
        t = self.page_graphs[n, bound]
        t["table"].copy_(self._page_lists(batch, t["table"].shape[1]))
        self._page_workspace(t)
        if graph and t["graph"] is None:
            t["graph"] = self._capture(lambda: self._pages_device_step(t))
            t["ws"] = self.page_ws  # whose address the graph holds
        if graph:
            t["graph"].replay()
        else:
            self._pages_device_step(t)

    def _pages_device_step(self, t):
        n = t["n"]
        torch.add(self.positions[:n], 1, out=t["lengths"])
        self._blocks(n, 0, attend=lambda i: self._attend_pages(i, t))
        self.logits_batch(range(n))
        self._call("gx_argmax_slots_step", self.ctx.ptr, self._vp(self.logit), self.cfg.vocab, n, self.cfg.vocab,
                   self._vp(self.next_id), self._vp(self.tokens), self._vp(self.positions))

    def free(self):
        for b in self.blocks:
            for k in ("qkv", "o", "gu", "down"):
                b[k].free()
        self.embd.free()
