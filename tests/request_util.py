"""Plain 64-bit forms of the operators on many requests' rows, and what their results may be off by."""
import math

import torch


def i32(values, device="cuda"):
    return torch.tensor(values, dtype=torch.int32, device=device)


def starts(new):
    return [sum(new[:i]) for i in range(len(new) + 1)]


def make_table(lens, page, seed, width=None, extra=0):
    """A block table whose pages lie in a random order, -1 behind each request's, and the number of pages (extra ones unused)."""
    gen = torch.Generator().manual_seed(seed)
    held = [-(-l // page) for l in lens]
    pages = torch.randperm(sum(held) + extra, generator=gen).tolist()
    width = max(max(held, default=0), 1) if width is None else width
    table = torch.full((len(lens), width), -1, dtype=torch.int32)
    at = 0
    for r, h in enumerate(held):
        table[r, :h] = torch.tensor(pages[at:at + h], dtype=torch.int32)
        at += h
    return table.cuda(), max(sum(held) + extra, 1)


def random_masks(new, seed, empty=0.0):
    """A row sees itself and random earlier tokens of its tree; a share of the rows sees no drafted token at all."""
    gen = torch.Generator().manual_seed(seed)
    out = []
    for n in new:
        for j in range(n):
            bits = 1 << j
            for i in range(j):
                if torch.rand(1, generator=gen).item() < 0.4:
                    bits |= 1 << i
            if torch.rand(1, generator=gen).item() < empty:
                bits = 0
            out.append(bits - (1 << 64) if bits >= 1 << 63 else bits)
    return torch.tensor(out, dtype=torch.int64, device="cuda")


def attend_ref(q, k, v, table, lens, new, mask, scale):
    """(out, tolerance) in 64 bits; k, v [pages, page, kv, D].

    The kernels sum scores and weights in f32 and may round a weight once to the rows' 16-bit type.  With u = half a step of that
    type: the result's own rounding is u |out|, the weights' is u sum w |v|, and a score's f32 error d (at most D steps of 2^-24 on
    sum |q k| scale, and the exponential's own) moves numerator and denominator by d each: 2 d sum w |v|."""
    T, H, D = q.shape
    page, kv = k.shape[1], k.shape[2]
    u = torch.finfo(q.dtype).eps / 2
    out = torch.zeros((T, H, D), dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    st = starts(new)
    kf, vf = k.double(), v.double()
    for r, (l, n) in enumerate(zip(lens, new)):
        if n == 0:
            continue
        p = torch.arange(l + n, device=q.device)
        pg = table[r, p // page].long()
        kr, vr = kf[pg, p % page], vf[pg, p % page]
        seen = torch.ones((n, l + n), dtype=torch.bool, device=q.device)
        if mask is None:
            seen[:, l:] = torch.ones((n, n), dtype=torch.bool, device=q.device).tril()
        else:
            seen[:, l:] = (mask[st[r]:st[r + 1], None] >> torch.arange(n, device=q.device)) & 1 == 1
        for h in range(H):
            qr = q[st[r]:st[r + 1], h].double()
            kk = kr[:, h // (H // kv)]
            # what a row does not see has no part in it, whatever it holds
            for j in range(n):
                s = seen[j]
                if not s.any():
                    continue
                ks, vs = kk[s], vr[s][:, h // (H // kv)]
                w = torch.softmax(ks @ qr[j] * scale, 0)
                o, mag = w @ vs, w @ vs.abs()
                d = D * 2.0 ** -24 * float((ks.abs() @ qr[j].abs()).max()) * abs(scale) + 2.0 ** -20
                out[st[r] + j, h] = o
                tol[st[r] + j, h] = u * o.abs() + (u + 2 * d) * mag + torch.finfo(q.dtype).smallest_normal * 2 * u
    return out, tol * 1.001


def lora_ref(x, A, B, scales, ranks, idx, base, residual=None):
    """(out, tolerance) in 64 bits: one rounding of the result to bf16, the f32 sums over K and rank (at most one step of 2^-23 per
    term of the sums of magnitudes), and x A^T carried to 2^-16 of its value between the two products."""
    out, mag = base.double().clone(), base.double().abs()
    for t, a in enumerate(idx.tolist()):
        if a < 0:
            continue
        r = A.shape[1] if ranks is None else int(ranks[a])
        low = A[a, :r].double() @ x[t].double()
        low_mag = A[a, :r].double().abs() @ x[t].double().abs()
        s = float(scales[a])
        out[t] += s * (B[a, :, :r].double() @ low)
        mag[t] += abs(s) * (B[a, :, :r].double().abs() @ (low_mag * x.shape[1] * 2.0 ** -23 + low.abs() * (2.0 ** -16 + r * 2.0 ** -23))) / 2.0 ** -22
    if residual is not None:
        out += residual.double()
        mag += residual.double().abs()
    return out, 2.0 ** -8 * out.abs() + 2.0 ** -22 * mag + 1e-38
