"""The 8-bit key-value format and the operators over it, restated in plain torch (64 bits where it matters)."""
import math

import torch

PAGE = 16
TOP = {"int8": 127.0, "fp8": 448.0}
FMTS = ("int8", "fp8")
# q heads, kv heads, head size: 32B, drafter, the small test models, MHA, a group that is no power of two, one KV head
LAYOUTS = [(64, 8, 128), (16, 8, 128), (4, 2, 64), (8, 8, 128), (10, 2, 64), (20, 1, 128)]


def encode(x, fmt):
    """uint8 codes and fp32 scales of the rows of fp32 ``x``, step for step as the format says."""
    scale = (x.abs().amax(-1, keepdim=True) / TOP[fmt]).clamp_min(2.0 ** -64)
    y = x / scale
    code = (y.round().clamp(-127, 127) + 128).to(torch.uint8) if fmt == "int8" else y.clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
    return code, scale.squeeze(-1)


def fields(pool, hd):
    p, h, _ = pool.shape
    return (pool[..., :PAGE * hd].view(p, h, PAGE, hd), pool[..., PAGE * hd:2 * PAGE * hd].view(p, h, PAGE, hd),
            pool[..., 2 * PAGE * hd:].view(torch.float32).view(p, h, PAGE, 2))


def values(pool, hd, fmt):
    """fp64 (k, v), each [pages, hkv, 16, hd]."""
    kc, vc, sc = fields(pool, hd)
    real = lambda c: c.double() - 128 if fmt == "int8" else c.contiguous().view(torch.float8_e4m3fn).double()
    return real(kc) * sc[..., :1].double(), real(vc) * sc[..., 1:].double()


class Cache:
    """Sequences of given lengths in shuffled pages of one pool (on the CPU); slots past a sequence's end and pages of no
    sequence are 0xff bytes, NaN in both formats, which nobody may see."""

    def __init__(self, lens, hkv, hd, fmt, seed=0, spare=3, k_amp=1.0, v_amp=1.0, k=None, v=None):
        g = torch.Generator().manual_seed(seed)
        need = [(n + PAGE - 1) // PAGE for n in lens]
        total = sum(need) + spare
        self.lens, self.hkv, self.hd, self.fmt = lens, hkv, hd, fmt
        self.pool = torch.full((total, hkv, 2 * PAGE * hd + 8 * PAGE), 0xFF, dtype=torch.uint8)
        self.bt = torch.full((len(lens), max(max(need), 1)), -1, dtype=torch.int32)
        order = torch.randperm(total, generator=g).tolist()
        kc, vc, sc = fields(self.pool, hd)
        for s, n in enumerate(lens):
            kk = (torch.randn(n, hkv, hd, generator=g) * k_amp) if k is None else k[s]
            vv = (torch.randn(n, hkv, hd, generator=g) * v_amp) if v is None else v[s]
            (ck, sk), (cv, sv) = encode(kk.float(), fmt), encode(vv.float(), fmt)
            for p in range(need[s]):
                page = order.pop()
                self.bt[s, p] = page
                m = min(PAGE, n - p * PAGE)
                at = slice(p * PAGE, p * PAGE + m)
                kc[page, :, :m], vc[page, :, :m] = ck[at].transpose(0, 1), cv[at].transpose(0, 1)
                sc[page, :, :m, 0], sc[page, :, :m, 1] = sk[at].transpose(0, 1), sv[at].transpose(0, 1)

    def rows(self, seq):
        """fp64 (k, v) of a sequence, [length, hkv, hd]."""
        k, v = values(self.pool, self.hd, self.fmt)
        n = self.lens[seq]
        ids = self.bt[seq, :(n + PAGE - 1) // PAGE].long()
        return tuple(t[ids].transpose(1, 2).reshape(-1, self.hkv, self.hd)[:n] for t in (k, v))


def attend(q, k, v, seen, hq, hkv):
    """fp64 result [hq, hd] of one row over the keys ``seen`` (bool), and how far a kernel may be from it.

    bf16 result: half a step, 2^-8 |o|.  Weights in fp16 (2^-11 each, both at the weight and at its sum) and scores in fp32 (their error,
    2^-17 of the sum of |q k| over 128 terms, moves a weight by as much relative to itself): (2^-10 + 2^-16 B) times the weighted mean of
    |v|.  Weights below fp16's normal range are off by 2^-25 of the largest contribution's scale: n 2^-24 max |v|."""
    hd, gq = q.shape[-1], hq // hkv
    n = int(seen.sum())
    if n == 0:
        return torch.zeros(hq, hd, dtype=torch.float64), torch.zeros(hq, hd, dtype=torch.float64)
    kk, vv = k[seen].transpose(0, 1), v[seen].transpose(0, 1)                    # [hkv, n, hd]
    qq = q.double().view(hkv, gq, hd)
    w = torch.softmax(qq @ kk.transpose(1, 2) / math.sqrt(hd), -1)
    big = (qq.abs() @ kk.abs().transpose(1, 2) / math.sqrt(hd)).amax(-1, keepdim=True)
    o = w @ vv
    tol = 2.0 ** -8 * o.abs() + (2.0 ** -10 + 2.0 ** -16 * big) * (w @ vv.abs()) + n * 2.0 ** -24 * vv.abs().amax((1, 2), keepdim=True)
    return o.reshape(hq, hd), tol.reshape(hq, hd)


def seen_keys(n_keys, pos, first=None, mask=None):
    """Keys of 0 .. n_keys - 1 that a row at ``pos`` sees; ``mask``: bits of the group's own slots, which begin at ``first``."""
    key = torch.arange(n_keys)
    ok = key <= pos
    if mask is not None:
        inside = key >= first
        bits = torch.tensor([bool((mask >> max(0, int(j) - first)) & 1) for j in key], dtype=torch.bool)
        ok = ok & (~inside | bits)
    return ok


def rotate(x, pos, inv_freq):
    """fp64 rotation of [heads, hd] by per-pair positions ``pos`` (number or [hd / 2])."""
    ang = torch.as_tensor(pos, dtype=torch.float64) * inv_freq.double()
    z = torch.complex(x[:, :x.shape[1] // 2].double(), x[:, x.shape[1] // 2:].double()) * torch.polar(torch.ones_like(ang), ang)
    return torch.cat([z.real, z.imag], -1)
