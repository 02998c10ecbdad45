"""The 8-bit key-value cache on the GPU against 64-bit restatements (``kv8_reference.py``)."""
import pytest
import torch

from agens_engine_b200.ops import attention as A
from agens_engine_b200.ops import basic
from agens_engine_b200.ops import kv8 as K

from tests.kv8_reference import FMTS, LAYOUTS, PAGE, TOP, Cache, attend, encode, fields, rotate, seen_keys, values

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def bf(x):
    return x.to(torch.bfloat16)


# --------------------------------------------------------------------------------------------------------------- store
def _store(hq, hkv, hd, fmt, pos, seq, bt, n_pages, qkv, **kw):
    """Runs the store over a pool of 0xff bytes; returns q, the pool (CPU) and the status."""
    pool = torch.full((n_pages, hkv, K.block_bytes(hd)), 0xFF, dtype=torch.uint8, device=DEV)
    q = torch.full((len(pos), hq * hd), 7.0, dtype=torch.bfloat16, device=DEV)
    st = K.rope_kvstore8(qkv.to(DEV), hq, hkv, hd, basic.rope_inv_freq(hd, 1e6, DEV), i32(pos), i32(seq), bt.to(DEV), pool, fmt, q, **kw)
    return q.cpu(), pool.cpu(), int(st.item())


def _check_stored(q, pool, hq, hkv, hd, fmt, pos, seq, bt, qkv, angle_pos):
    inv = basic.rope_inv_freq(hd, 1e6, "cpu")
    kc, vc, sc = fields(pool, hd)
    k, v = values(pool, hd, fmt)
    touched = torch.zeros(pool.shape[0], PAGE, dtype=torch.bool)
    for i, (p, s) in enumerate(zip(pos, seq)):
        page, slot = int(bt[s, p // PAGE]), p % PAGE
        touched[page, slot] = True
        row = qkv[i].view(hq + 2 * hkv, hd)
        ref = rotate(row[:hq + hkv].float(), angle_pos(i), inv)
        # sines and cosines in fp32 (two steps of 2^-24 each), two products and a sum, times at most |x| + |y|
        half = hd // 2
        mag = row[:hq + hkv].float().abs().double()
        slack = 2.0 ** -21 * (mag[:, :half] + mag[:, half:]).repeat(1, 2)
        assert bool(((q[i].view(hq, hd).double() - ref[:hq]).abs() <= 2.0 ** -8 * ref[:hq].abs() + slack[:hq]).all()), i
        rk, sk = ref[hq:], slack[hq:].amax(-1, keepdim=True)
        amax = rk.abs().amax(-1, keepdim=True)
        scale = sc[page, :, slot, 0].double().unsqueeze(-1)
        assert bool(((scale - amax / TOP[fmt]).abs() <= 2.0 ** -22 * scale + sk / TOP[fmt]).all()), i
        # int8: half a step of scale; e4m3: half a step of 2^-4 relative, 2^-10 of the scale below its normal numbers
        step = scale * 0.5 if fmt == "int8" else 2.0 ** -4 * rk.abs() + 2.0 ** -10 * scale
        assert bool(((k[page, :, slot] - rk).abs() <= step * (1 + 2.0 ** -10) + 2 * sk).all()), i
        code, vs = encode(row[hq + hkv:].float(), fmt)                     # bf16 inputs and one division: bit for bit
        assert torch.equal(vc[page, :, slot], code) and torch.equal(sc[page, :, slot, 1], vs), i
    # every slot that no row names is as it was
    assert bool((kc.transpose(1, 2)[~touched] == 0xFF).all()) and bool((vc.transpose(1, 2)[~touched] == 0xFF).all())
    assert bool((sc.view(torch.int32).transpose(1, 2)[~touched] == -1).all())


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("hq,hkv,hd", LAYOUTS)
def test_store_rotates_and_quantises(hq, hkv, hd, fmt):
    torch.manual_seed(hq + hd)
    pos, seq = [0, 15, 16, 17, 40, 1048570, 99999], [0, 0, 0, 0, 1, 2, 1]
    bt = torch.full((3, 65537), -1, dtype=torch.int32)
    bt[0, 0], bt[0, 1], bt[1, 2], bt[1, 99999 // PAGE], bt[2, 1048570 // PAGE] = 5, 0, 2, 6, 3
    wide = bf(torch.randn(len(pos), (hq + 2 * hkv) * hd + 24))
    qkv = wide[:, 8:8 + (hq + 2 * hkv) * hd]                                  # rows of a wider buffer
    q, pool, st = _store(hq, hkv, hd, fmt, pos, seq, bt, 7, qkv)
    assert st == 0
    _check_stored(q, pool, hq, hkv, hd, fmt, pos, seq, bt, qkv, lambda i: float(pos[i]))


@pytest.mark.parametrize("n", [1, 3, 33, 257])
def test_store_of_a_chunk_with_its_own_rotary_positions(n):
    """Rotary positions that differ from the slots (one axis), and three axes."""
    torch.manual_seed(n)
    hq, hkv, hd, start = 10, 2, 64, 21
    pos, seq = list(range(start, start + n)), [0] * n
    pages = (start + n + PAGE - 1) // PAGE
    bt = torch.randperm(pages).to(torch.int32).view(1, -1)
    qkv = bf(torch.randn(n, (hq + 2 * hkv) * hd))
    rp = torch.randint(0, 40000, (n,), dtype=torch.int32)
    q, pool, st = _store(hq, hkv, hd, "int8", pos, seq, bt, pages, qkv, rope_pos=rp.to(DEV))
    assert st == 0
    _check_stored(q, pool, hq, hkv, hd, "int8", pos, seq, bt, qkv, lambda i: float(rp[i]))
    p3 = torch.randint(0, 5000, (3, n), dtype=torch.int32)
    axis = basic.mrope_pair_axis(hd, (12, 10, 10))
    q, pool, st = _store(hq, hkv, hd, "fp8", pos, seq, bt, pages, qkv, rope_pos3=p3.to(DEV), pair_axis=axis.to(DEV))
    assert st == 0
    _check_stored(q, pool, hq, hkv, hd, "fp8", pos, seq, bt, qkv, lambda i: p3[:, i].double()[axis.long()])


@pytest.mark.parametrize("fmt", FMTS)
def test_store_of_unusual_rows(fmt):
    """Zeros, the smallest and largest numbers, infinities and NaN; a row's neighbours do not notice."""
    hq, hkv, hd = 2, 1, 64
    qkv = bf(torch.randn(7, (hq + 2 * hkv) * hd))
    tiny, huge = 2.0 ** -126, 3e38
    qkv[0, hq * hd:] = 0
    qkv[1, hq * hd:] = bf(torch.randn(2 * hd)) * tiny
    qkv[2, hq * hd:] *= 1e36
    qkv[3, -5] = float("inf")
    qkv[4, -64] = float("nan")
    qkv[5, -1] = huge
    pos = list(range(7))
    bt = torch.tensor([[1]], dtype=torch.int32)
    q, pool, st = _store(hq, hkv, hd, fmt, pos, [0] * 7, bt, 2, qkv)
    assert st == 0
    k, v = (t[1, 0, :7] for t in values(pool, hd, fmt))
    sc = fields(pool, hd)[2][1, 0, :7]
    assert bool((k[0] == 0).all()) and bool((v[0] == 0).all()) and bool((sc[0] == 2.0 ** -64).all())
    assert bool((v[1].abs() <= 2.0 ** -64).all()) and bool((sc[1] == 2.0 ** -64).all())       # below the format's smallest step
    assert bool(torch.isnan(v[3]).all()) and bool(torch.isnan(v[4]).all())
    for r in (2, 5, 6):
        code, s = encode(qkv[r, (hq + hkv) * hd:].float().view(1, hd), fmt)
        assert torch.equal(fields(pool, hd)[1][1, 0, r], code[0]) and float(sc[r, 1]) == float(s[0])
    assert bool(torch.isfinite(k[[0, 1, 3, 4, 6]]).all())


def test_store_skips_and_reports_what_is_out_of_range():
    hq, hkv, hd = 4, 2, 64
    pos, seq = [3, 16, 20, 33, 5, -1, 2 ** 31 - 1, 4], [0, 0, 0, 0, 1, 0, 0, 0]
    bt = torch.tensor([[2, 9, -1]], dtype=torch.int32)          # 16, 20: no such page; 33: no page; sequence 1: none; slots without a table entry
    qkv = bf(torch.randn(len(pos), (hq + 2 * hkv) * hd))
    q, pool, st = _store(hq, hkv, hd, "int8", pos, seq, bt, 4, qkv)
    assert st == 4
    good = [0, 7]
    touched = torch.zeros(4, PAGE, dtype=torch.bool)
    touched[2, 3] = touched[2, 4] = True
    assert bool((pool[[0, 1, 3]] == 0xFF).all())
    _check_stored(q[good], pool, hq, hkv, hd, "int8", [pos[i] for i in good], [0, 0], bt, qkv[good], lambda i: float(pos[good[i]]))


@pytest.mark.parametrize("hq,hkv,hd,n", [(6, 1, 128, 297), (64, 8, 128, 301), (5, 3, 64, 650)])
def test_store_of_many_tokens_some_of_them_nowhere(hq, hkv, hd, n):
    """An odd number of tokens, where blocks take two; slots 96 to 111 have no page, one token no sequence."""
    pos, seq = list(range(n)), [0] * n
    pages = (n + PAGE - 1) // PAGE
    bt = torch.randperm(pages).to(torch.int32).view(1, -1)
    bt[0, 6] = pages
    seq[n - 2] = 1
    qkv = bf(torch.randn(n, (hq + 2 * hkv) * hd))
    q, pool, st = _store(hq, hkv, hd, "int8", pos, seq, bt, pages, qkv)
    assert st == 4
    good = [i for i in range(n) if i // PAGE != 6 and i != n - 2]
    _check_stored(q[good], pool, hq, hkv, hd, "int8", [pos[i] for i in good], [0] * len(good), bt, qkv[good], lambda i: float(good[i]))


# ---------------------------------------------------------------------------------------------------------------- read
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("hkv,hd,n", [(8, 128, 1), (2, 64, 16), (1, 128, 17), (3, 64, 100), (2, 128, 333)])
def test_read_gives_the_values_of_the_pages(hkv, hd, n, fmt):
    c = Cache([n], hkv, hd, fmt, seed=n, k_amp=3.0)
    pages = c.bt[0]
    got = K.kv_read8(c.pool.to(DEV), fmt, pages.to(DEV), n_tokens=n).cpu()
    k, v = values(c.pool, hd, fmt)
    live = (torch.arange(pages.numel() * PAGE) < n).view(-1, 1, PAGE, 1)
    for i, t in enumerate((k, v)):
        # code times scale rounded to fp32, then to bf16: what torch gives for the same two steps
        ref = torch.where(live, t[pages.long()].float(), torch.zeros(())).to(torch.bfloat16)
        assert torch.equal(got[:, i], ref)
    # every slot, whatever it holds; the same page twice; an output that the caller gives
    twice = torch.cat([pages, pages[:1]])
    out = torch.full((twice.numel(), 2, hkv, PAGE, hd), 3.0, dtype=torch.bfloat16, device=DEV)
    st = torch.zeros(1, dtype=torch.int32, device=DEV)
    assert K.kv_read8(c.pool.to(DEV), fmt, twice.to(DEV), out=out, status=st) is out and int(st.item()) == 0
    assert torch.equal(out[0].cpu().view(torch.int16), out[-1].cpu().view(torch.int16))
    assert torch.equal(torch.nan_to_num(out[:-1].cpu()) * live.unsqueeze(1), got)


def test_read_reports_pages_that_are_not_there():
    c = Cache([40], 2, 64, "int8")
    st = torch.zeros(1, dtype=torch.int32, device=DEV)
    got = K.kv_read8(c.pool.to(DEV), "int8", i32([int(c.bt[0, 0]), 99, -1]), n_tokens=48, status=st)
    assert int(st.item()) == 4 and bool((got[1:] == 0).all()) and bool((got[0] != 0).any())
    st.zero_()
    got = K.kv_read8(c.pool.to(DEV), "int8", i32([int(c.bt[0, 0]), 99, -1]), n_tokens=16, status=st)      # pages past the end are not looked at
    assert int(st.item()) == 0 and bool((got[1:] == 0).all())


# -------------------------------------------------------------------------------------------------------------- attend
def _groups(lens, new):
    """Index tensors of one group of ``new[s]`` rows at the end of every sequence (lengths count them)."""
    pos, seq, g0, gc = [], [], [], []
    for s, (n, r) in enumerate(zip(lens, new)):
        g0.append(len(pos)); gc.append(r)
        pos += list(range(n - r, n)); seq += [s] * r
    return pos, seq, g0, gc


def _attend(c, q, hq, pos, seq, g0, gc, mask=None, pool=None, **kw):
    st = torch.zeros(1, dtype=torch.int32, device=DEV)
    out = K.attn_decode8(q.to(DEV), c.pool.to(DEV) if pool is None else pool, c.fmt, c.bt.to(DEV), i32(g0), i32(gc), i32(pos), i32(seq), hq, c.hkv,
                         c.hd, tree_mask=None if mask is None else i32(mask), status=st, **kw)
    assert int(st.item()) == 0
    return out.cpu()


def _check_attend(c, q, hq, out, pos, seq, g0, gc, mask=None):
    kv = [c.rows(s) for s in range(len(c.lens))]
    for first, cnt in zip(g0, gc):
        for t in range(first, first + cnt):
            k, v = kv[seq[t]]
            seen = seen_keys(k.shape[0], pos[t], pos[first], None if mask is None else mask[t] & 0xFFFFFFFF)
            ref, tol = attend(q[t].view(hq, c.hd), k, v, seen, hq, c.hkv)
            off = (out[t].view(hq, c.hd).double() - ref).abs()
            assert bool((off <= tol).all()), (t, float((off - tol).max()))


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("hq,hkv,hd", LAYOUTS)
def test_attend_decode_and_verify(hq, hkv, hd, fmt):
    lens, new = [1, 16, 17, 130, 300, 777, 40], [1, 1, 2, 4, 8, 1, 3]
    c = Cache(lens, hkv, hd, fmt, seed=hq, k_amp=2.0)
    pos, seq, g0, gc = _groups(lens, new)
    q = bf(torch.randn(len(pos), hq * hd))
    out = _attend(c, q, hq, pos, seq, g0, gc)
    _check_attend(c, q, hq, out, pos, seq, g0, gc)
    # a row's bits do not depend on its company: every row as a decode step of its own
    pool = c.pool.to(DEV)
    for t in range(len(pos)):
        assert torch.equal(_attend(c, q[t:t + 1], hq, pos[t:t + 1], seq[t:t + 1], [0], [1], pool=pool)[0], out[t]), t


@pytest.mark.parametrize("fmt", FMTS)
def test_attend_over_a_long_cache(fmt):
    hq, hkv, hd = 16, 2, 128
    lens, new = [5003, 4096], [1, 5]
    c = Cache(lens, hkv, hd, fmt, seed=9, k_amp=4.0, v_amp=0.01)
    pos, seq, g0, gc = _groups(lens, new)
    q = bf(torch.randn(len(pos), hq * hd))
    out = _attend(c, q, hq, pos, seq, g0, gc)
    _check_attend(c, q, hq, out, pos, seq, g0, gc)
    pool = c.pool.to(DEV)
    for t in range(len(pos)):
        assert torch.equal(_attend(c, q[t:t + 1], hq, pos[t:t + 1], seq[t:t + 1], [0], [1], pool=pool)[0], out[t]), t


@pytest.mark.parametrize("hq,hkv,hd", [(64, 8, 128), (10, 2, 64)])
def test_attend_tree_masks_and_rows_that_see_nothing(hq, hkv, hd):
    """Trees over the group's own slots; groups at the very start of a sequence, where an empty mask leaves a row nothing."""
    lens, new = [8, 67, 300, 32, 5], [8, 6, 3, 32, 5]
    c = Cache(lens, hkv, hd, "int8", seed=4)
    pos, seq, g0, gc = _groups(lens, new)
    g = torch.Generator().manual_seed(2)
    mask = []
    for cnt in gc:
        m = [1]
        for r in range(1, cnt):
            m.append(m[int(torch.randint(0, r, (1,), generator=g))] | (1 << r))
        mask += m
    mask[2] = mask[g0[4]] = mask[g0[4] + 3] = 0               # nothing at all: these sequences begin with their group
    mask = [x - (1 << 32) if x >= 1 << 31 else x for x in mask]
    q = bf(torch.randn(len(pos), hq * hd))
    out = _attend(c, q, hq, pos, seq, g0, gc, mask)
    _check_attend(c, q, hq, out, pos, seq, g0, gc, mask)
    assert bool((out[[2, g0[4], g0[4] + 3]] == 0).all())


def test_attend_rows_without_keys_padding_and_strides():
    """Position -1 (a padded row of a batch) gives zeros; rows of no group and the columns beside a strided output stay."""
    hq, hkv, hd = 8, 2, 128
    c = Cache([20, 50], hkv, hd, "fp8", seed=1)
    pos, seq = [19, -1, 49, 48], [0, 0, 1, 1]
    q = bf(torch.randn(4, hq * hd + 64))[:, 16:16 + hq * hd]
    wide = torch.full((6, hq * hd + 16), 5.0, dtype=torch.bfloat16, device=DEV)
    out = wide[:4, 8:8 + hq * hd]
    K.attn_decode8(q.to(DEV), c.pool.to(DEV), "fp8", c.bt.to(DEV), i32([0, 1, 2, 3]), i32([1, 1, 1, 0]), i32(pos), i32(seq), hq, hkv, hd, out=out)
    got = wide.cpu()
    assert bool((got[:4, :8] == 5).all()) and bool((got[:4, 8 + hq * hd:] == 5).all()) and bool((got[3:] == 5).all())
    assert bool((got[1, 8:-8] == 0).all())
    rows = got[:4, 8:8 + hq * hd]
    for t in (0, 2):
        k, v = c.rows(seq[t])
        ref, tol = attend(q[t].reshape(hq, hd), k, v, seen_keys(k.shape[0], pos[t]), hq, hkv)
        assert bool(((rows[t].view(hq, hd).double() - ref).abs() <= tol).all())


@pytest.mark.parametrize("split", [16, 48, 64, 2048])
def test_attend_split_sizes_and_a_workspace_of_the_caller(split):
    """Any split gives the result within the bound; what lies in the workspace before or behind its part does not matter."""
    hq, hkv, hd = 16, 2, 64
    lens, new = [1, 47, 49, 1003], [1, 1, 2, 7]
    c = Cache(lens, hkv, hd, "fp8", seed=split)
    pos, seq, g0, gc = _groups(lens, new)
    q = bf(torch.randn(len(pos), hq * hd))
    need = K.part_floats(len(pos), hq, hd, c.bt.shape[1] * PAGE, split)
    part = torch.full((need + 64,), float("nan"), device=DEV)
    out = _attend(c, q, hq, pos, seq, g0, gc, split_keys=split, part=part)
    _check_attend(c, q, hq, out, pos, seq, g0, gc)
    assert bool(torch.isnan(part[need:]).all())
    # groups in another order, one group a call, and more groups than a warp has lanes
    order = [3, 1, 0, 2]
    again = _attend(c, q, hq, pos, seq, [g0[i] for i in order], [gc[i] for i in order], split_keys=split)
    assert torch.equal(again, out)
    many = _attend(c, q, hq, pos, seq, g0 * 17 + list(range(len(pos))), gc * 17 + [1] * len(pos), split_keys=split)
    assert torch.equal(many, out)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("lens,new,split", [([1500, 1400, 1450, 901], [6] * 4, 128), ([40 + 83 * i % 600 for i in range(40)], [1] * 40, 64)])
def test_attend_work_of_many_groups_heads_and_splits(lens, new, split, fmt):
    """Several times as much as runs at once: what works on one head or group goes on with the next one."""
    hq, hkv, hd = 64, 8, 128
    c = Cache(lens, hkv, hd, fmt, seed=split, k_amp=2.0)
    pos, seq, g0, gc = _groups(lens, new)
    q = bf(torch.randn(len(pos), hq * hd))
    out = _attend(c, q, hq, pos, seq, g0, gc, split_keys=split)
    _check_attend(c, q, hq, out, pos, seq, g0, gc)
    pool = c.pool.to(DEV)
    for t in range(len(pos)):
        assert torch.equal(_attend(c, q[t:t + 1], hq, pos[t:t + 1], seq[t:t + 1], [0], [1], pool=pool, split_keys=split)[0], out[t]), t


def test_attend_more_groups_than_a_warp_has_lanes():
    hq, hkv, hd = 4, 2, 64
    lens = [1 + 37 * i % 190 for i in range(75)]
    new = [1 + i % min(5, n) for i, n in enumerate(lens)]
    c = Cache(lens, hkv, hd, "int8", seed=1)
    pos, seq, g0, gc = _groups(lens, new)
    gc[40] = 0                                                # rows of no group: not written
    q = bf(torch.randn(len(pos), hq * hd))
    out = torch.full((len(pos), hq * hd), 9.0, dtype=torch.bfloat16, device=DEV)
    got = _attend(c, q, hq, pos, seq, g0, gc, split_keys=32, out=out)
    _check_attend(c, q, hq, got, pos, seq, g0, gc)
    assert bool((got[g0[40]:g0[41]] == 9).all())


def test_attend_calls_that_run_at_the_same_time():
    """Two streams and two graphs, captured on one stream and replayed on two, none with a workspace of the caller."""
    hq, hkv, hd = 64, 8, 128
    c = Cache([3000, 2500], hkv, hd, "int8", seed=5)
    pool, bt = c.pool.to(DEV), c.bt.to(DEV)
    q = [bf(torch.randn(2, hq * hd)).to(DEV) for _ in range(4)]
    args = (bt, i32([0, 1]), i32([1, 1]), i32([2999, 2499]), i32([0, 1]), hq, hkv, hd)
    st = torch.zeros(1, dtype=torch.int32, device=DEV)
    run = lambda i, o: K.attn_decode8(q[i], pool, "int8", *args, split_keys=64, status=st, out=o)
    want = [run(i, None).clone() for i in range(4)]
    out = [torch.zeros_like(want[0]) for _ in range(4)]
    streams = [torch.cuda.Stream() for _ in range(4)]
    graphs = []
    torch.cuda.synchronize()
    for i in (2, 3):
        with torch.cuda.stream(streams[0]):
            run(i, out[i])
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=streams[0]):
            run(i, out[i])
        graphs.append(g)
    for _ in range(20):
        for o in out:
            o.zero_()
        torch.cuda.synchronize()
        for i in range(4):
            with torch.cuda.stream(streams[i]):
                if i < 2:
                    run(i, out[i])
                else:
                    graphs[i - 2].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
    assert int(st.item()) == 0


def test_attend_refuses_positions_past_max_ctx():
    hq, hkv, hd = 4, 2, 64
    c = Cache([600, 600], hkv, hd, "int8")
    q = bf(torch.randn(2, hq * hd)).to(DEV)
    out = torch.full((2, hq * hd), 9.0, dtype=torch.bfloat16, device=DEV)
    st = torch.zeros(1, dtype=torch.int32, device=DEV)
    K.attn_decode8(q, c.pool.to(DEV), "int8", c.bt.to(DEV), i32([0, 1]), i32([1, 1]), i32([599, 255]), i32([0, 1]), hq, hkv, hd, split_keys=256, max_ctx=512,
                   status=st, out=out)
    assert int(st.item()) == 4 and bool((out[0] == 9).all())
    k, v = c.rows(1)
    ref, tol = attend(q[1].cpu().view(hq, hd), k, v, seen_keys(600, 255), hq, hkv)
    assert bool(((out[1].cpu().view(hq, hd).double() - ref).abs() <= tol).all())


def test_attend_rows_that_others_see_may_be_nan():
    """A row of the group whose V is NaN: rows whose mask leaves it out do not notice."""
    hq, hkv, hd = 8, 1, 64
    for fmt in FMTS:
        c = Cache([40], hkv, hd, fmt, seed=2)
        fields(c.pool, hd)[2][int(c.bt[0, 2]), 0, 5, :] = float("nan")       # token 37
        pos, seq, g0, gc = _groups([40], [4])                                  # rows 36 .. 39
        q = bf(torch.randn(4, hq * hd))
        out = _attend(c, q, hq, pos, seq, g0, gc, [1, 3, 5, 0b1010])
        assert bool(torch.isfinite(out[[0, 2]]).all()) and bool(torch.isnan(out[[1, 3]]).all())
        k, v = c.rows(0)
        for t, m in ((0, 1), (2, 5)):
            ref, tol = attend(q[t].view(hq, hd), k, v, seen_keys(40, pos[t], 36, m), hq, hkv)
            assert bool(((out[t].view(hq, hd).double() - ref).abs() <= tol).all())


@pytest.mark.parametrize("fmt", FMTS)
def test_attend_scales_of_every_size(fmt):
    """V rows of very different sizes, a heavy key whose V is zero (it takes weight and adds nothing), tiny and huge V, large scores."""
    hq, hkv, hd = 8, 1, 128
    g = torch.Generator().manual_seed(5)
    n = 210
    k = [torch.randn(n, hkv, hd, generator=g) for _ in range(4)]
    v = [torch.randn(n, hkv, hd, generator=g) for _ in range(4)]
    v[0] *= torch.exp(4 * torch.randn(n, 1, 1, generator=g))
    v[1][7] = 0
    v[2] *= 1e-17
    v[3] *= 1e30
    q = bf(torch.randn(4, hq * hd, generator=g))
    k[1][7] = 6 * q[1].float().view(hq, hd).mean(0) * hq ** 0.5
    k[3] *= 20
    c = Cache([n] * 4, hkv, hd, fmt, k=k, v=v)
    pos, seq, g0, gc = _groups([n] * 4, [1] * 4)
    out = _attend(c, q, hq, pos, seq, g0, gc)
    _check_attend(c, q, hq, out, pos, seq, g0, gc)
    assert bool((out[2].float().abs() > 0).any())


def test_attend_a_non_finite_row_shows_and_stays_where_it_is():
    hq, hkv, hd = 16, 2, 64
    c = Cache([100, 100], hkv, hd, "int8", seed=6)
    sc = fields(c.pool, hd)[2]
    sc[int(c.bt[0, 3]), 1, 4, 1] = float("nan")              # V of token 52 of sequence 0, KV head 1
    pos, seq, g0, gc = [51, 52, 99, 99], [0, 0, 0, 1], [0, 1, 2, 3], [1, 1, 1, 1]
    q = bf(torch.randn(4, hq * hd))
    out = _attend(c, q, hq, pos, seq, g0, gc).view(4, hq, hd)
    assert bool(torch.isfinite(out[[0, 3]]).all()) and bool(torch.isfinite(out[1:3, :8]).all()) and bool(torch.isnan(out[1:3, 8:]).all())


def test_attend_skips_and_reports_what_is_out_of_range():
    hq, hkv, hd = 8, 2, 64
    c = Cache([40, 40, 40], hkv, hd, "int8", seed=3)
    bt = c.bt.clone()
    bt[1, 0] = 10 ** 6                                        # a page that is not there: its keys are left out
    q = bf(torch.randn(6, hq * hd)).to(DEV)
    out = torch.full((6, hq * hd), 9.0, dtype=torch.bfloat16, device=DEV)
    st = torch.zeros(1, dtype=torch.int32, device=DEV)
    run = lambda pos, seq, g0, gc: K.attn_decode8(q, c.pool.to(DEV), "int8", bt.to(DEV), i32(g0), i32(gc), i32(pos), i32(seq), hq, hkv, hd, status=st, out=out)
    run([39, 39, 39, 39, 39, 39], [0, 1, 2, 0, 0, 0], [0, 1, 2], [1, 1, 1])
    assert int(st.item()) == 4
    got = out.cpu()
    for t, s in ((0, 0), (1, 1), (2, 2)):
        k, v = c.rows(s)
        seen = seen_keys(40, 39)
        seen[:16] &= s != 1
        ref, tol = attend(q[t].cpu().view(hq, hd), k, v, seen, hq, hkv)
        assert bool(((got[t].view(hq, hd).double() - ref).abs() <= tol).all()), t
    # groups past the rows, sequences and tables that there are: left out, their neighbours not
    for pos, seq, g0, gc in (([39] * 6, [0] * 6, [0, 5], [1, 2]), ([39] * 6, [0] * 6, [0, -1], [1, 1]), ([39] * 6, [0, 3] + [0] * 4, [0, 1], [1, 1]),
                             ([39, 48] + [39] * 4, [0] * 6, [0, 1], [1, 1]), ([39, 2 ** 31 - 1] + [39] * 4, [0] * 6, [0, 1], [1, 1])):
        st.zero_()
        out.fill_(9.0)
        run(pos, seq, g0, gc)
        assert int(st.item()) == 4 and torch.equal(out[0].cpu(), got[0]) and bool((out[1:] == 9).all())


# ------------------------------------------------------------------------------------------- the operators as they are used
@pytest.mark.parametrize("fmt", FMTS)
def test_store_then_attend_then_read_then_prefill(fmt):
    """A conversation: a chunk is written and read back for the prefill attention, then single tokens are written and attended."""
    torch.manual_seed(11)
    hq, hkv, hd, T, steps = 16, 2, 128, 200, 5
    n = T + steps
    bt = torch.randperm(20)[:(n + PAGE - 1) // PAGE].to(torch.int32).view(1, -1).to(DEV)
    pool = K.make_pool(20, hkv, hd, DEV)
    inv = basic.rope_inv_freq(hd, 1e6, DEV)
    qkv = bf(torch.randn(n, (hq + 2 * hkv) * hd)).to(DEV)
    st = torch.zeros(1, dtype=torch.int32, device=DEV)
    at = lambda a, b: torch.arange(a, b, dtype=torch.int32, device=DEV)
    zeros = torch.zeros(n, dtype=torch.int32, device=DEV)
    q = torch.empty(n, hq * hd, dtype=torch.bfloat16, device=DEV)
    K.rope_kvstore8(qkv[:T], hq, hkv, hd, inv, at(0, T), zeros, bt, pool, fmt, q[:T], status=st)
    stage = K.kv_read8(pool, fmt, bt[0], n_tokens=T, status=st)
    o = A.attn_prefill_tc(q[:T], stage, at(0, stage.shape[0]).view(1, -1), 0, 0, hq, hkv, status=st)
    outs = [o]
    for t in range(T, n):
        K.rope_kvstore8(qkv[t:t + 1], hq, hkv, hd, inv, at(t, t + 1), zeros, bt, pool, fmt, q[t:t + 1], status=st)
        outs.append(K.attn_decode8(q[t:t + 1], pool, fmt, bt, zeros[:1], i32([1]), at(t, t + 1), zeros, hq, hkv, hd, status=st))
    assert int(st.item()) == 0
    out = torch.cat(outs).cpu()
    k, v = (x[bt[0].cpu().long()].transpose(1, 2).reshape(-1, hkv, hd) for x in values(pool.cpu(), hd, fmt))
    for t in [0, 1, 15, 63, 199] + list(range(T, n)):
        ref, tol = attend(q[t].cpu().view(hq, hd), k, v, seen_keys(k.shape[0], t), hq, hkv)
        if t < T:
            # the prefill kernel works on K, V and weights in bf16: 2^-8 of each, K's through the scores
            big = (q[t].cpu().double().view(hkv, -1, hd).abs() @ k[:t + 1].abs().permute(1, 2, 0)).amax() / hd ** 0.5
            tol = tol + (3 + float(big)) * 2.0 ** -8 * v[:t + 1].abs().amax()
        assert bool(((out[t].view(hq, hd).double() - ref).abs() <= tol).all()), t


def test_captured_replayed_and_on_a_stream_of_its_own():
    """A step (store, attend) in a CUDA graph gives what the eager calls give, replay after replay, from another stream."""
    torch.manual_seed(12)
    hq, hkv, hd, fmt = 16, 8, 128, "int8"
    lens = [33, 700, 5]
    c = Cache(lens, hkv, hd, fmt, seed=8)
    pool, bt = c.pool.to(DEV), c.bt.to(DEV)
    inv = basic.rope_inv_freq(hd, 1e6, DEV)
    qkv = bf(torch.randn(3, (hq + 2 * hkv) * hd)).to(DEV)
    pos, seq = i32([n - 1 for n in lens]), i32([0, 1, 2])
    g0, gc, st = i32([0, 1, 2]), i32([1, 1, 1]), torch.zeros(1, dtype=torch.int32, device=DEV)
    q, out = torch.empty(3, hq * hd, dtype=torch.bfloat16, device=DEV), torch.empty(3, hq * hd, dtype=torch.bfloat16, device=DEV)

    def step(p, o):
        K.rope_kvstore8(qkv, hq, hkv, hd, inv, pos, seq, bt, p, fmt, q, status=st)
        K.attn_decode8(q, p, fmt, bt, g0, gc, pos, seq, hq, hkv, hd, status=st, out=o)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(pool, out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step(pool, out)
    for trial in range(3):
        qkv.copy_(bf(torch.randn(3, (hq + 2 * hkv) * hd)))
        pos.sub_(trial)                                       # the positions are read on the device
        want_pool, want = pool.clone(), torch.empty_like(out)
        step(want_pool, want)
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(pool, want_pool)
    assert int(st.item()) == 0
