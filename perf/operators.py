"""The operators of the 8-bit key-value cache as cases that can be timed and checked.

Three operators (``agens_engine_b200.ops.kv8``): ``store`` rotates the q and k of fused qkv rows and writes k and v into
8-bit pages, ``attend`` is the attention of new tokens over such pages, ``read`` gives pages back in bf16.  ``run`` makes
the engine's calls where ``own`` is true and computes the plain form in torch otherwise; ``exact`` restates the definition
in 64 bits.

A pool is uint8 ``[pages, kv heads, 32 * hd + 128]``: of every page (16 tokens) and KV head the K codes ``[16][hd]``, the V
codes ``[16][hd]`` and 16 pairs of fp32 scales (K, V).  A row's scale is amax / 127 ("int8": codes -127 .. 127, stored with
128 added) or amax / 448 ("fp8": e4m3), at least 2^-64.  A stored row stands for code * scale.

Head layouts are those of the engine's configurations and tests (64 / 8, 16 / 8 and 16 / 2 heads of 128, 4 / 2 of 64),
lengths those of its serving: decode steps of one to 64 conversations, verify blocks of up to eight rows, prefill chunks of up
to 2048 rows, contexts up to 131072 tokens.
"""
from __future__ import annotations

import functools
import math

import torch

own = False

DEV = "cuda:0"
PAGE = 16
THETA = 1e6
MIN_SCALE = 2.0 ** -64


# ---------------------------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # the new token of one conversation, 32B heads: the smallest store, bound by latency
        dict(name="store_1token_int8", op="store", fmt="int8", hq=64, hkv=8, hd=128, seqs=1, rows=1, pos0=5003, axes=1),
        # a decode step of 48 conversations of the companion drafter
        dict(name="store_48seqs_fp8", op="store", fmt="fp8", hq=16, hkv=8, hd=128, seqs=48, rows=1, pos0=2101, axes=1),
        # a chunk of an image prompt (three-axis positions), odd length and start, heads of 64
        dict(name="store_chunk_333_fp8", op="store", fmt="fp8", hq=4, hkv=2, hd=64, seqs=1, rows=333, pos0=77, axes=3),
        # a 2048-row prefill chunk after 6144 tokens, 32B heads
        dict(name="store_chunk_2048_int8", op="store", fmt="int8", hq=64, hkv=8, hd=128, seqs=1, rows=2048, pos0=6144, axes=1),
        # one new token of a short conversation, 32B heads
        dict(name="attend_1seq_700_int8", op="attend", fmt="int8", hq=64, hkv=8, hd=128, seqs=1, rows=1, ctx=700),
        # a decode step of 24 conversations of different lengths, 32B heads
        dict(name="attend_24seqs_fp8", op="attend", fmt="fp8", hq=64, hkv=8, hd=128, seqs=24, rows=1, ctx=4001),
        # verify blocks of six drafted rows (a tree) of four conversations
        dict(name="attend_verify_tree_int8", op="attend", fmt="int8", hq=64, hkv=8, hd=128, seqs=4, rows=6, ctx=9001),
        # a decode step of 64 conversations, a model with heads of 64 and two q heads per KV head
        dict(name="attend_64seqs_hd64_int8", op="attend", fmt="int8", hq=4, hkv=2, hd=64, seqs=64, rows=1, ctx=2500),
        # one new token after 131072 tokens: a long document
        dict(name="attend_long_int8", op="attend", fmt="int8", hq=64, hkv=8, hd=128, seqs=1, rows=1, ctx=131072),
        # the pages of a short context handed to the prefill attention of the next chunk
        dict(name="read_1000_fp8", op="read", fmt="fp8", hq=64, hkv=8, hd=128, tokens=1000),
        # the same at the end of a medium one, drafter heads
        dict(name="read_6151_int8", op="read", fmt="int8", hq=16, hkv=2, hd=128, tokens=6151),
        # and of a long one
        dict(name="read_65536_int8", op="read", fmt="int8", hq=64, hkv=8, hd=128, tokens=65536),
    ]


HEADS = [(64, 8, 128), (64, 8, 128), (16, 8, 128), (16, 2, 128), (8, 8, 128), (4, 2, 64)]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    hq, hkv, hd = rng.choice(HEADS)
    base = dict(fmt=rng.choice(["int8", "fp8"]), hq=hq, hkv=hkv, hd=hd)
    op = rng.choice(["store", "store", "attend", "attend", "attend", "read"])
    if op == "store":
        if rng.random() < 0.5:
            return dict(op=op, **base, seqs=_log(rng, 1, 64), rows=1, pos0=_log(rng, 1, 100000), axes=1)
        return dict(op=op, **base, seqs=1, rows=_log(rng, 2, 2048), pos0=rng.choice([0, _log(rng, 1, 30000)]), axes=rng.choice([1, 1, 3]))
    if op == "attend":
        rows = rng.choice([1, 1, rng.randint(2, 8)])
        if rng.random() < 0.5:
            return dict(op=op, **base, seqs=_log(rng, 1, 64 if rows == 1 else 8), rows=rows, ctx=_log(rng, 1, 3800))
        return dict(op=op, **base, seqs=1, rows=rows, ctx=_log(rng, 500, 100000 if rows == 1 else 50000))
    return dict(op=op, **base, tokens=_log(rng, 1, 65000))


# ------------------------------------------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _lengths(case):
    """Tokens in the cache of every conversation: from ctx down to about half of it."""
    s = case["seqs"]
    return [max(1, case["ctx"] - (i * case["ctx"]) // (2 * s)) for i in range(s)]


def _encode(x, fmt):
    """Codes (uint8) and scales (fp32) of the rows of fp32 ``x``."""
    top = 127.0 if fmt == "int8" else 448.0
    scale = (x.abs().amax(-1, keepdim=True) / top).clamp_min(MIN_SCALE)
    y = x / scale
    if fmt == "int8":
        code = (y.round().clamp(-127, 127) + 128).to(torch.uint8)
    else:
        code = y.clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
    return code, scale.squeeze(-1)


def _fields(pool, hd):
    """K codes, V codes [pages, hkv, 16, hd] and scales [pages, hkv, 16, 2] of a pool, as views."""
    p, h, _ = pool.shape
    return (pool[..., :PAGE * hd].view(p, h, PAGE, hd), pool[..., PAGE * hd:2 * PAGE * hd].view(p, h, PAGE, hd),
            pool[..., 2 * PAGE * hd:].view(torch.float32).view(p, h, PAGE, 2))


def _filled_pool(g, n_pages, hkv, hd, fmt):
    """Pages as a model leaves them: normal values, K with a few channels several times larger, heads of different sizes."""
    pool = torch.empty(n_pages, hkv, 2 * PAGE * hd + 128, dtype=torch.uint8, device=DEV)
    kc, vc, sc = _fields(pool, hd)
    amp = torch.exp(0.5 * torch.randn(2, hkv, 1, 1, device=DEV, generator=g))
    chan = torch.where(torch.rand(hkv, 1, hd, device=DEV, generator=g) < 0.03, 4.0, 1.0)
    step = max(1, (64 << 20) // (hkv * PAGE * hd))
    for p0 in range(0, n_pages, step):
        n = min(step, n_pages - p0)
        for i, dst in ((0, kc), (1, vc)):
            x = torch.randn(n, hkv, PAGE, hd, device=DEV, generator=g) * amp[i]
            c, s = _encode(x * chan if i == 0 else x, fmt)
            dst[p0:p0 + n] = c
            sc[p0:p0 + n, :, :, i] = s
    return pool


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _table(g, lens):
    """A block table over shuffled pages, -1 where a conversation has none, and the number of pages."""
    need = [(n + PAGE - 1) // PAGE for n in lens]
    total = sum(need)
    order = torch.randperm(total, device=DEV, generator=g).to(torch.int32)
    bt = torch.full((len(lens), max(need)), -1, dtype=torch.int32, device=DEV)
    at = 0
    for i, n in enumerate(need):
        bt[i, :n] = order[at:at + n]
        at += n
    return bt, total


def prepare(case, seed):
    g = _gen(seed)
    hq, hkv, hd, fmt = case["hq"], case["hkv"], case["hd"], case["fmt"]
    st = dict(op=case["op"], fmt=fmt, hq=hq, hkv=hkv, hd=hd, status=torch.zeros(1, dtype=torch.int32, device=DEV))
    if case["op"] == "store":
        n, seqs, rows = case["seqs"] * case["rows"], case["seqs"], case["rows"]
        pos = [case["pos0"] + (7 * s) % 53 + r for s in range(seqs) for r in range(rows)]
        seq = [s for s in range(seqs) for _ in range(rows)]
        # pages of the touched part only: what lies before is not read by this operator
        width = max(pos) // PAGE + 1
        touched = sorted({(s, p // PAGE) for s, p in zip(seq, pos)})
        order = torch.randperm(len(touched), generator=torch.Generator().manual_seed(int(seed))).tolist()
        bt = torch.full((seqs, width), -1, dtype=torch.int32)
        bt[[s for s, _ in touched], [p for _, p in touched]] = torch.tensor(order, dtype=torch.int32)
        i = torch.arange(0, hd // 2, dtype=torch.float64)
        st.update(qkv=torch.randn(n, (hq + 2 * hkv) * hd, device=DEV, generator=g).to(torch.bfloat16),
                  inv_freq=(THETA ** (-2.0 * i / hd)).to(torch.float32).to(DEV), tok_pos=_i32(pos), tok_seq=_i32(seq),
                  block_table=bt.to(DEV), pages=_i32(order), pool=_filled_pool(g, len(touched), hkv, hd, fmt),
                  q_out=torch.empty(n, hq * hd, dtype=torch.bfloat16, device=DEV), pos3=None, pair_axis=None)
        if case["axes"] == 3:
            # a picture of 32 columns: the time stands still, rows and columns count on
            at = st["tok_pos"]
            st["pos3"] = torch.stack([torch.full_like(at, case["pos0"]), case["pos0"] + (at - case["pos0"]) // 32,
                                      case["pos0"] + (at - case["pos0"]) % 32]).contiguous()
            st["pair_axis"] = (torch.arange(hd // 2, device=DEV) % 3).to(torch.uint8)
        return st
    if case["op"] == "attend":
        lens, rows = _lengths(case), case["rows"]
        bt, total = _table(g, [n + rows - 1 for n in lens])
        n_tok = len(lens) * rows
        st.update(q=(1.5 * torch.randn(n_tok, hq * hd, device=DEV, generator=g)).to(torch.bfloat16), block_table=bt,
                  pool=_filled_pool(g, total, hkv, hd, fmt), grp_tok0=_i32(list(range(0, n_tok, rows))), grp_cnt=_i32([rows] * len(lens)),
                  tok_pos=_i32([n - 1 + r for n in lens for r in range(rows)]), tok_seq=_i32([s for s in range(len(lens)) for _ in range(rows)]),
                  rows=rows, tree_mask=None, out=torch.empty(n_tok, hq * hd, dtype=torch.bfloat16, device=DEV))
        if rows > 1:
            # drafted trees: every row hangs on an earlier one and sees its ancestors
            c = torch.Generator().manual_seed(int(seed))
            masks = []
            for _ in lens:
                m = [1]
                for r in range(1, rows):
                    m.append(m[int(torch.randint(0, r, (1,), generator=c))] | (1 << r))
                masks += m
            st["tree_mask"] = _i32(masks)
        return st
    n = case["tokens"]
    bt, total = _table(g, [n])
    st.update(pool=_filled_pool(g, total, hkv, hd, fmt), pages=bt[0].contiguous(), tokens=n)
    return st


# --------------------------------------------------------------------------------------------------------- plain form
def _values(pool, hd, fmt, pages):
    """fp32 values [pages, 2, hkv, 16, hd] of the named pages."""
    kc, vc, sc = _fields(pool, hd)
    pages = pages.long()
    code = torch.stack([kc[pages], vc[pages]], 1)
    code = code.float() - 128.0 if fmt == "int8" else code.view(torch.float8_e4m3fn).float()
    return code * sc[pages].permute(0, 3, 1, 2).unsqueeze(-1)


def _plain_store(st):
    hq, hkv, hd, fmt = st["hq"], st["hkv"], st["hd"], st["fmt"]
    n, half = st["qkv"].shape[0], hd // 2
    x = st["qkv"].float().view(n, hq + 2 * hkv, hd)
    # angles in 64 bits: a 32-bit product of a far position loses the angle itself
    pos = st["tok_pos"].double().unsqueeze(1) if st["pos3"] is None else st["pos3"].double()[st["pair_axis"].long()].t()
    ang = pos * st["inv_freq"].double()
    c, s = torch.cos(ang).float().unsqueeze(1), torch.sin(ang).float().unsqueeze(1)
    lo, hi = x[:, :hq + hkv, :half], x[:, :hq + hkv, half:]
    rot = torch.cat([lo * c - hi * s, hi * c + lo * s], -1)
    q = rot[:, :hq].reshape(n, hq * hd).to(torch.bfloat16)
    kc, vc, sc = _fields(st["pool"], hd)
    at = st["tok_pos"].long()
    page, slot = st["block_table"][st["tok_seq"].long(), at // PAGE].long(), at % PAGE
    k_code, k_scale = _encode(rot[:, hq:], fmt)
    v_code, v_scale = _encode(x[:, hq + hkv:], fmt)
    kc[page, :, slot] = k_code
    vc[page, :, slot] = v_code
    sc[page, :, slot] = torch.stack([k_scale, v_scale], -1)
    return q, _values(st["pool"], hd, fmt, st["pages"]).to(torch.bfloat16)


def _plain_attend(st):
    hq, hkv, hd, rows = st["hq"], st["hkv"], st["hd"], st["rows"]
    bt = st["block_table"]
    seqs, width = bt.shape
    kv = _values(st["pool"], hd, st["fmt"], bt.clamp_min(0).reshape(-1)).view(seqs, width, 2, hkv, PAGE, hd)
    kv = kv.permute(2, 0, 3, 1, 4, 5).reshape(2, seqs * hkv, width * PAGE, hd)
    q = st["q"].float().view(seqs, rows, hkv, hq // hkv, hd).transpose(1, 2).reshape(seqs * hkv, rows * (hq // hkv), hd)
    s = torch.bmm(q, kv[0].transpose(1, 2)) / math.sqrt(hd)
    key = torch.arange(width * PAGE, device=DEV)
    pos = st["tok_pos"].view(seqs, rows, 1)
    seen = key <= pos
    if st["tree_mask"] is not None:
        inside = key - pos[:, :1]
        bit = (st["tree_mask"].view(seqs, rows, 1) >> inside.clamp(0, 31)) & 1
        seen = seen & ((inside < 0) | (bit == 1))
    seen = seen.view(seqs, 1, rows, 1, width * PAGE).expand(seqs, hkv, rows, hq // hkv, width * PAGE).reshape(s.shape)
    s = s.masked_fill(~seen, -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    o = torch.bmm(p, kv[1]) / p.sum(-1, keepdim=True)
    return o.view(seqs, hkv, rows, hq // hkv, hd).transpose(1, 2).reshape(seqs * rows, hq * hd).to(torch.bfloat16)


def _plain_read(st):
    v = _values(st["pool"], st["hd"], st["fmt"], st["pages"])
    slot = torch.arange(st["pages"].numel() * PAGE, device=DEV).view(-1, 1, 1, PAGE, 1)
    return torch.where(slot < st["tokens"], v, 0.0).to(torch.bfloat16)


# ---------------------------------------------------------------------------------------------------------------- run
@functools.lru_cache(None)
def _kv8():
    from agens_engine_b200.ops import kv8
    return kv8


def run(state):
    st = state
    if own:
        K = _kv8()
        if st["op"] == "store":
            K.rope_kvstore8(st["qkv"], st["hq"], st["hkv"], st["hd"], st["inv_freq"], st["tok_pos"], st["tok_seq"], st["block_table"],
                            st["pool"], st["fmt"], st["q_out"], rope_pos3=st["pos3"], pair_axis=st["pair_axis"], status=st["status"])
            return st["q_out"], K.kv_read8(st["pool"], st["fmt"], st["pages"], status=st["status"])
        if st["op"] == "attend":
            return K.attn_decode8(st["q"], st["pool"], st["fmt"], st["block_table"], st["grp_tok0"], st["grp_cnt"], st["tok_pos"],
                                  st["tok_seq"], st["hq"], st["hkv"], st["hd"], tree_mask=st["tree_mask"], status=st["status"],
                                  out=st["out"])
        return K.kv_read8(st["pool"], st["fmt"], st["pages"], n_tokens=st["tokens"], status=st["status"])
    if st["op"] == "store":
        return _plain_store(st)
    return _plain_attend(st) if st["op"] == "attend" else _plain_read(st)


def work(case):
    hq, hkv, hd = case["hq"], case["hkv"], case["hd"]
    row8 = hkv * (2 * hd + 8)                       # one token in the cache: codes and scales of K and V
    row16 = hkv * 2 * hd * 2                        # the same in bf16
    if case["op"] == "store":
        n = case["seqs"] * case["rows"]
        pos = [case["pos0"] + (7 * s) % 53 for s in range(case["seqs"])]
        slots = sum((p + case["rows"] - 1) // PAGE - p // PAGE + 1 for p in pos) * PAGE
        # rows in, rotated q and quantised k, v out; then the touched pages read back
        return {"bytes": n * ((hq + 2 * hkv) * hd * 2 + hq * hd * 2 + row8) + slots * (row8 + row16),
                "flops": n * ((hq + hkv) * hd * 3 + 2 * hkv * hd * 3) + slots * 2 * hkv * hd}
    if case["op"] == "attend":
        keys = sum(n + case["rows"] - 1 for n in _lengths(case))
        seen = sum(n + r for n in _lengths(case) for r in range(case["rows"]))
        n_tok = case["seqs"] * case["rows"]
        return {"bytes": keys * row8 + n_tok * hq * hd * 4, "flops": seen * hq * hd * 4}
    slots = (case["tokens"] + PAGE - 1) // PAGE * PAGE
    return {"bytes": case["tokens"] * row8 + slots * row16, "flops": case["tokens"] * 2 * hkv * hd}


# -------------------------------------------------------------------------------------------------- the 64-bit results
def _real(code, fmt):
    """What a stored byte stands for, in 64 bits."""
    b = code.to(torch.int64)
    if fmt == "int8":
        return (b - 128).double()
    e, m = (b >> 3) & 15, (b & 7).double()
    mag = torch.where(e == 0, m * 2.0 ** -9, (1.0 + m / 8.0) * torch.exp2((e - 7).double()))
    return torch.where(b >= 128, -mag, mag)


def _quantised(x, fmt):
    """Rows of 64-bit ``x`` as the format holds them."""
    top = 127.0 if fmt == "int8" else 448.0
    scale = torch.clamp(x.abs().amax(-1, keepdim=True) / top, min=MIN_SCALE)
    y = x / scale
    if fmt == "int8":
        return torch.clamp(torch.round(y), -127, 127) * scale
    # e4m3: eight steps between powers of two, the smallest step 2^-9
    step = torch.exp2(torch.clamp(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -40))), min=-6.0) - 3.0)
    return torch.clamp(torch.round(y / step) * step, -448, 448) * scale


def exact(case, seed):
    st = prepare(case, seed)
    hq, hkv, hd, fmt = case["hq"], case["hkv"], case["hd"], case["fmt"]
    kb, vb = PAGE * hd, 2 * PAGE * hd

    def rows_of(page_ids):
        raw = st["pool"].index_select(0, page_ids.long())
        sc = raw[..., vb:].contiguous().view(torch.float32).double().view(-1, hkv, PAGE, 2)
        k = _real(raw[..., :kb], fmt).view(-1, hkv, PAGE, hd) * sc[..., :1]
        v = _real(raw[..., kb:vb], fmt).view(-1, hkv, PAGE, hd) * sc[..., 1:]
        return k, v

    if case["op"] == "store":
        x = st["qkv"].double().view(-1, hq + 2 * hkv, hd)
        n = x.shape[0]
        pos = st["tok_pos"].double().view(n, 1).expand(n, hd // 2)
        if st["pos3"] is not None:
            pos = torch.gather(st["pos3"].double().t(), 1, st["pair_axis"].long().view(1, -1).expand(n, -1))
        turn = torch.polar(torch.ones_like(pos), pos * st["inv_freq"].double())
        z = torch.complex(x[:, :hq + hkv, :hd // 2], x[:, :hq + hkv, hd // 2:]) * turn.view(n, 1, -1)
        rot = torch.cat([z.real, z.imag], -1)
        k, v = rows_of(torch.arange(st["pool"].shape[0], device=DEV))
        new_k, new_v = _quantised(rot[:, hq:], fmt), _quantised(x[:, hq + hkv:], fmt)
        where = st["tok_pos"].long()
        page = st["block_table"][st["tok_seq"].long(), where // PAGE].long()
        for h in range(hkv):
            k[:, h][page, where % PAGE] = new_k[:, h]
            v[:, h][page, where % PAGE] = new_v[:, h]
        return rot[:, :hq].reshape(n, -1), torch.stack([k, v], 1)[st["pages"].long()]
    if case["op"] == "attend":
        out = torch.empty(st["q"].shape[0], hq, hd, dtype=torch.float64, device=DEV)
        for s in range(case["seqs"]):
            ids = st["block_table"][s]
            k, v = rows_of(ids[ids >= 0])
            k, v = (t.transpose(0, 1).reshape(hkv, -1, hd) for t in (k, v))
            for r in range(case["rows"]):
                i = s * case["rows"] + r
                first, last = int(st["tok_pos"][s * case["rows"]]), int(st["tok_pos"][i])
                keep = torch.ones(last + 1, dtype=torch.bool, device=DEV)
                if st["tree_mask"] is not None:
                    m = int(st["tree_mask"][i])
                    keep[first:] = torch.tensor([bool((m >> j) & 1) for j in range(last + 1 - first)], device=DEV)
                q = st["q"][i].double().view(hkv, hq // hkv, hd)
                w = torch.softmax(q @ k[:, :last + 1][:, keep].transpose(1, 2) / math.sqrt(hd), -1)
                out[i] = (w @ v[:, :last + 1][:, keep]).reshape(hq, hd)
        return out.view(-1, hq * hd)
    k, v = rows_of(st["pages"])
    both = torch.stack([k, v], 1)
    live = (torch.arange(both.shape[0] * PAGE, device=DEV) < case["tokens"]).view(-1, 1, 1, PAGE, 1)
    return both * live
