"""A nanochat-shaped language model whose attention blocks are DISM layers (hard path).

Plain torch everywhere except the sequence mixer: bias-free q/k/v/output projections, rotary position
embedding (base 100000) and a parameter-free RMS norm on q and k, pre-norm residual blocks, a 4x MLP with
squared ReLU, untied embedding and unembedding (the shape of the reference's nanochat GPT:
nanochat/nanochat/gpt.py:42-43,77-80,101-102,142-150,161-166,284-291).  The mixer replaces the attention
call (gpt.py:109-130) by `voc_dism` and adds what the reference's DISM module adds per layer: readout
projections sq/sk with SiLU (dism_v3/python/flash_dism/module.py:118-119,151-159), two codebooks [H,V,D]
initialised silu(N(0,1)) and a per-head log_sel_tau ~ U(-4,4) whose softplus is the weight coefficient
(module.py:125-131,376-380).  Every sequence runs hard: the operator's gradient reaches the model through
sq, sk, v and tau, as in the reference's hard training rows.

Chosen layers can be gated delta layers instead, as in the reference's hybrid (dism_v3/python/flash_dism/hybrid_gdn.py), which can also
decode one token at a time from a state, and both branches of a block can pass through residual dropout.
"""
import math
import operator

import torch
import torch.nn as nn
import torch.nn.functional as F


def rms(x, eps=1e-6):
    return x * torch.rsqrt(x.float().square().mean(-1, keepdim=True) + eps).to(x.dtype)


def rotary(x, cos, sin):
    """x [B,N,H,D]; cos, sin [N,1,D/2]."""
    a, b = x[..., : x.size(-1) // 2], x[..., x.size(-1) // 2:]
    return torch.cat((a * cos + b * sin, b * cos - a * sin), -1)


class DismLayer(nn.Module):
    def __init__(self, width, heads, head_dim, readout_dim=32, vocab_size=512):
        super().__init__()
        self.heads, self.head_dim, self.readout_dim = heads, head_dim, readout_dim
        self.c_q = nn.Linear(width, heads * head_dim, bias=False)
        self.c_k = nn.Linear(width, heads * head_dim, bias=False)
        self.c_v = nn.Linear(width, heads * head_dim, bias=False)
        self.c_proj = nn.Linear(heads * head_dim, width, bias=False)
        self.sq_proj = nn.Linear(width, heads * readout_dim, bias=False)
        self.sk_proj = nn.Linear(width, heads * readout_dim, bias=False)
        self.q_vocab = nn.Parameter(F.silu(torch.randn(heads, vocab_size, head_dim)))
        self.k_vocab = nn.Parameter(F.silu(torch.randn(heads, vocab_size, head_dim)))
        self.log_sel_tau = nn.Parameter(torch.empty(heads).uniform_(-4, 4))

    def forward(self, x, cos, sin, hard):
        from flash_dism import voc_dism
        b, n, _ = x.shape
        split = lambda t, d: t.view(b, n, self.heads, d)
        q, k, v = split(self.c_q(x), self.head_dim), split(self.c_k(x), self.head_dim), split(self.c_v(x), self.head_dim)
        q, k = rms(rotary(q, cos, sin)), rms(rotary(k, cos, sin))
        sq, sk = F.silu(split(self.sq_proj(x), self.readout_dim)), F.silu(split(self.sk_proj(x), self.readout_dim))
        tau = F.softplus(self.log_sel_tau.float())
        out = voc_dism(q, k, sq, sk, v, self.q_vocab, self.k_vocab, tau, direction=None, hard=hard)
        return self.c_proj(out.flatten(2))


class DeltaLayer(nn.Module):
    """Gated delta mixer: unit queries and keys, values, a decay -exp(log_rate) softplus(a + bias) and a write strength sigmoid(b) per
    head, and an output RMS norm with a SiLU gate (rates uniform in [0, 16), steps log-uniform in [1e-3, 1e-1], as such layers are
    usually started).  No positions enter: the decay orders the sequence."""

    def __init__(self, width, heads, head_dim):
        super().__init__()
        self.heads, self.head_dim = heads, head_dim
        self.c_q, self.c_k, self.c_v, self.c_gate = (nn.Linear(width, heads * head_dim, bias=False) for _ in range(4))
        self.c_decay, self.c_write = (nn.Linear(width, heads, bias=False) for _ in range(2))
        self.c_proj = nn.Linear(heads * head_dim, width, bias=False)
        self.log_rate = nn.Parameter(torch.empty(heads).uniform_(1e-3, 16).log())
        step = torch.exp(torch.empty(heads).uniform_(math.log(1e-3), math.log(1e-1)))
        self.decay_bias = nn.Parameter(step + torch.log(-torch.expm1(-step)))

    def operands(self, x):
        split = lambda t: t.view(*t.shape[:-1], self.heads, self.head_dim)
        q, k = (rms(split(c(x))) * self.head_dim ** -.5 for c in (self.c_q, self.c_k))
        decay = -self.log_rate.float().exp() * F.softplus(self.c_decay(x).float() + self.decay_bias.float())
        return q, k, split(self.c_v(x)), decay, torch.sigmoid(self.c_write(x).float())

    def finish(self, out, x):
        return self.c_proj((rms(out) * F.silu(self.c_gate(x)).view_as(out)).flatten(-2))

    def forward(self, x, cos=None, sin=None, hard=None):
        from flash_dism import gated_delta_rule
        return self.finish(gated_delta_rule(*self.operands(x)), x)

    def prefill(self, x, state=None):
        """Whole sequences [B,N,width]; returns the output and the state [B,H,D,D] after the last position."""
        from flash_dism import gated_delta_rule
        out, state = gated_delta_rule(*self.operands(x), initial_state=state, output_final_state=True)
        return self.finish(out, x), state

    def step(self, x, state, slots=None):
        """One token per row [B,width]; `state` is updated in place."""
        from flash_dism import gated_delta_step
        return self.finish(gated_delta_step(*self.operands(x), state, slots=slots), x)


class Block(nn.Module):
    def __init__(self, width, heads, head_dim, mixer=DismLayer):
        super().__init__()
        self.mixer = mixer(width, heads, head_dim)
        self.c_fc = nn.Linear(width, 4 * width, bias=False)
        self.c_out = nn.Linear(4 * width, width, bias=False)

    def mlp(self, x):
        return self.c_out(F.relu(self.c_fc(rms(x))).square())

    def forward(self, x, cos, sin, hard, p=0., seed=None, site=0):
        if not p:
            x = x + self.mixer(rms(x), cos, sin, hard)
            return x + self.mlp(x)
        from flash_dism import dropout_add
        x = dropout_add(self.mixer(rms(x), cos, sin, hard), x, p, seed, site=site)
        return dropout_add(self.mlp(x), x, p, seed, site=site + 1)


class DismLM(nn.Module):
    """depth x (mixer + MLP); logits over `vocab` tokens; cross-entropy when targets are given.

    `delta_layers` names the blocks (by index) whose mixer is a DeltaLayer, the others are DISM layers.  `dropout` is the probability of
    residual dropout while training; its masks follow the buffer `dropout_seed`, int64 (key, offset), whose offset the program
    advances once a step (model.dropout_seed[1] += 1, after the backward pass) and which checkpoints hold.  Data-parallel replicas, whose
    buffers may be one rank's, each set `dropout_rank` to draw masks of their own.  A model of delta layers only also runs
    from states: prefill() a prompt, then step() token by token."""

    def __init__(self, depth=20, width=1280, heads=10, head_dim=128, vocab=65536, rope_base=100000., delta_layers=(), dropout=0.,
                 dropout_rank=0):
        super().__init__()
        self.heads, self.head_dim, self.rope_base, self.dropout, self.dropout_rank = heads, head_dim, rope_base, dropout, dropout_rank
        self.embed = nn.Embedding(vocab, width)
        delta_layers = {operator.index(i) for i in delta_layers}
        if not delta_layers <= set(range(depth)):
            raise ValueError(f'delta_layers must name blocks 0 to {depth - 1}')
        self.blocks = nn.ModuleList(Block(width, heads, head_dim, DeltaLayer if i in delta_layers else DismLayer) for i in range(depth))
        if dropout:
            self.register_buffer('dropout_seed', torch.randint(0, 1 << 62, (2,)) * torch.tensor([1, 0]))
        self.unembed = nn.Linear(width, vocab, bias=False)

    def _load_from_state_dict(self, state_dict, prefix, *rest):
        # weights go from a model with dropout to one without and back
        if self.dropout:
            state_dict.setdefault(prefix + 'dropout_seed', self.dropout_seed)
        else:
            state_dict.pop(prefix + 'dropout_seed', None)
        super()._load_from_state_dict(state_dict, prefix, *rest)

    def angles(self, n, device, dtype):
        inverse = 1. / self.rope_base ** (torch.arange(0, self.head_dim, 2, device=device, dtype=torch.float32) / self.head_dim)
        phase = torch.outer(torch.arange(n, device=device, dtype=torch.float32), inverse)
        return phase.cos()[:, None].to(dtype), phase.sin()[:, None].to(dtype)

    def forward(self, tokens, targets=None):
        b, n = tokens.shape
        x = rms(self.embed(tokens))
        cos, sin = self.angles(n, x.device, x.dtype)
        hard = torch.ones(b, self.heads, dtype=torch.bool, device=x.device)
        p, seed = (self.dropout, self.dropout_seed) if self.dropout and self.training else (0., None)
        for index, block in enumerate(self.blocks):
            x = block(x, cos, sin, hard, p, seed, 2 * (index + self.dropout_rank * len(self.blocks)))
        logits = self.unembed(rms(x))
        if targets is None:
            return logits
        return F.cross_entropy(logits.float().view(-1, logits.size(-1)), targets.reshape(-1))

    def _recurrent(self, states):
        if not all(isinstance(block.mixer, DeltaLayer) for block in self.blocks):
            raise NotImplementedError('DISM layers have no state to decode from; only a model of delta layers steps token by token')
        if states is not None and len(states) != len(self.blocks):
            raise ValueError('one state per block required')

    @torch.no_grad()
    def prefill(self, tokens, states=None):
        """tokens [B,N] -> (logits of the last position [B,vocab], one FP32 state [B,H,D,D] per block); `states` continues earlier ones."""
        self._recurrent(states)
        x, after = rms(self.embed(tokens)), []
        for index, block in enumerate(self.blocks):
            y, state = block.mixer.prefill(rms(x), None if states is None else states[index])
            x, after = x + y, after + [state]
            x = x + block.mlp(x)
        return self.unembed(rms(x[:, -1])), after

    @torch.no_grad()
    def step(self, tokens, states, slots=None):
        """One token per row, tokens [B] -> logits [B,vocab]; the states are updated in place (`slots`: int32 [B], each row's state)."""
        self._recurrent(states)
        x = rms(self.embed(tokens))
        for block, state in zip(self.blocks, states):
            x = x + block.mixer.step(rms(x), state, slots)
            x = x + block.mlp(x)
        return self.unembed(rms(x))
