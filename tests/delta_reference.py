"""The gated delta rule token by token in 64 bits, differentiable: what the tests compare the kernels with."""
import numpy as np
import torch


def sequences(q, k, v, g, beta, scale, initial=None, starts=None):
    """[B,N,HK,D] q, k, [B,N,H,DV] v, [B,N,H] gates -> output and last states, in the operands' own (64-bit) type.
    starts: document starts of a pack (rows of no document are zeros)."""
    if starts is None:
        spans = [(b, 0, v.shape[1]) for b in range(v.shape[0])]
    else:
        spans = [(0, a, b) for a, b in zip(starts, starts[1:])]
    groups = v.shape[2] // q.shape[2]
    q, k = (x.repeat_interleave(groups, 2) for x in (q, k))
    rows = {}
    finals = []
    for index, (b, begin, end) in enumerate(spans):
        s = torch.zeros(v.shape[2], q.shape[3], v.shape[3], dtype=v.dtype, device=v.device) if initial is None else initial[index]
        for t in range(begin, end):
            s = torch.exp(g[b, t])[:, None, None] * s
            u = beta[b, t][:, None] * (v[b, t] - torch.einsum('hij,hi->hj', s, k[b, t]))
            s = s + k[b, t][:, :, None] * u[:, None, :]
            rows[b, t] = scale * torch.einsum('hij,hi->hj', s, q[b, t])
        finals.append(s)
    nothing = torch.zeros_like(v[0, 0]) if v.shape[1] else None
    out = [torch.stack([rows.get((b, t), nothing) for t in range(v.shape[1])]) if v.shape[1] else v[b] for b in range(v.shape[0])]
    return torch.stack(out), torch.stack(finals)


def operands(seed, b, n, key_heads, heads, d, dv, gates=torch.bfloat16, decay=.5, device='cpu'):
    """Unit queries and keys (bf16), values, log decays of about -decay and write strengths."""
    g = torch.Generator().manual_seed(seed)
    unit = lambda: torch.nn.functional.normalize(torch.randn(b, n, key_heads, d, generator=g), dim=-1).bfloat16()
    q, k = unit(), unit()
    v = torch.randn(b, n, heads, dv, generator=g).bfloat16()
    log_decay = (-decay * torch.rand(b, n, heads, generator=g)).to(gates)
    beta = torch.sigmoid(torch.randn(b, n, heads, generator=g)).to(gates)
    return [x.to(device) for x in (q, k, v, log_decay, beta)]


def philox(count, key, offset, site):
    """The 16-bit numbers of Philox4x32-10 blocks, eight to a block (numpy, 64-bit products)."""
    word, shift = np.uint64(0xFFFFFFFF), np.uint64(32)
    blocks = np.arange((count + 7) // 8, dtype=np.uint64)
    x = [blocks & word, np.full_like(blocks, site), np.full_like(blocks, offset & 0xFFFFFFFF), np.full_like(blocks, (offset >> 32) & 0xFFFFFFFF)]
    for turn in range(10):
        k0, k1 = (np.uint64(((key >> s) + turn * w) & 0xFFFFFFFF) for s, w in ((0, 0x9E3779B9), (32, 0xBB67AE85)))
        a, b = x[0] * np.uint64(0xD2511F53), x[2] * np.uint64(0xCD9E8D57)
        x = [(b >> shift) ^ x[1] ^ k0, b & word, (a >> shift) ^ x[3] ^ k1, a & word]
    return np.stack(x, 1).astype(np.uint32).view(np.uint16).reshape(-1)[:count]
