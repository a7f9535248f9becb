"""The MXFP4 and mixture-of-experts operators in 64 bits (torch, CPU), from their
definitions: the oracle of ``xpu_kernels.mxfp4`` and ``xpu_kernels.moe``."""

import torch

GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def scale_width(k):
    return (k + 511) // 512 * 16


def quantize(x):
    """(codes uint8 [.., K/2], scales uint8 [.., scale_width(K)])."""
    x = x.detach().cpu().double()
    k = x.shape[-1]
    b = x.reshape(*x.shape[:-1], k // 32, 32)
    amax = b.abs().amax(-1)
    bad = ~torch.isfinite(b).all(-1)
    mant, ex = torch.frexp(torch.where(bad | (amax == 0), 1.0, amax))
    e = torch.where(amax == 0, -127, (ex - 1 - 2).clamp(-127, 127))
    v = torch.where(bad[..., None], 0.0, b) / torch.ldexp(torch.ones(()).double(), e)[..., None]
    a = v.abs()
    # nearest on the grid; on a tie the even code (0, 1, 2, 4 among the pairs' halves)
    code = torch.zeros_like(a, dtype=torch.uint8)
    for c in range(1, 8):
        mid = (GRID[c - 1] + GRID[c]) / 2
        code += ((a > mid) | ((a == mid) & (c % 2 == 0))).to(torch.uint8)
    code |= torch.signbit(b).to(torch.uint8) << 3
    code = code.reshape(*x.shape[:-1], k)
    codes = code[..., 0::2] | (code[..., 1::2] << 4)
    scales = torch.full((*x.shape[:-1], scale_width(k)), 127, dtype=torch.uint8)
    scales[..., :k // 32] = torch.where(bad, 255, e + 127).to(torch.uint8)
    return codes, scales


def dequantize(codes, scales):
    codes, scales = codes.cpu(), scales.cpu()
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).long()
    k = c.shape[-1]
    v = torch.tensor(GRID, dtype=torch.float64)[c & 7]
    v = torch.where(c >= 8, -v, v)
    s = scales[..., :k // 32].long()
    f = torch.where(s == 255, float("nan"), torch.ldexp(torch.ones(()).double(), s - 127))
    return v * f.repeat_interleave(32, -1)


def sort(ids, n_experts):
    """(order, position, rows, offsets) as int32."""
    ids = ids.cpu()
    flat = ids.reshape(-1).tolist()
    key = [e if 0 <= e < n_experts else n_experts for e in flat]
    order = sorted(range(len(flat)), key=lambda s: (key[s], s))
    position = [0] * len(flat)
    for i, s in enumerate(order):
        position[s] = i
    offsets = [sum(1 for k in key if k < e) for e in range(n_experts + 1)]
    top = ids.shape[1]
    t = torch.int32
    return (torch.tensor(order, dtype=t), torch.tensor(position, dtype=t).reshape(ids.shape),
            torch.tensor([s // top for s in order], dtype=t), torch.tensor(offsets, dtype=t))


def grouped(xq, wq, rows, offsets):
    """sum_k xq[rows[i], k] wq[e, n, k] in 64 bits, zeros for the rows of no expert."""
    y = torch.zeros(rows.numel(), wq.shape[1], dtype=torch.float64)
    off = offsets.tolist()
    for e in range(wq.shape[0]):
        r = slice(off[e], off[e + 1])
        y[r] = xq[rows[r].long()] @ wq[e].t()
    return y
