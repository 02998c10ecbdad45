"""Prefill of the dense model over 8-bit pages: chunks below and above the prefill attention's least size."""
import pytest
import torch

from agens_engine_b200.models import config as C
from agens_engine_b200.models import oracle as O
from agens_engine_b200.models.dense import DenseModel
from agens_engine_b200.ops import kv8 as K

pytestmark = pytest.mark.gpu
FMTS = ["int8", "fp8"]


@pytest.fixture(scope="module")
def tiny():
    cfg = C.oracle_tiny()
    return cfg, O.random_weights(cfg, seed=0)


def test_short_chunks_take_no_workspace_but_the_steps(tiny):
    """A chunk of 9 to 63 rows: where its context is one split it needs no workspace, and elsewhere the steps' own, in pieces of rows; the
    size of the block table costs nothing.  The bits are those of a model whose workspace holds the chunk at once."""
    cfg, ow = tiny
    kw = dict(max_ctx=131072, n_pages=80, kv_cache="int8")
    m, wide = DenseModel.from_oracle(ow, max_seqs=1, **kw), DenseModel.from_oracle(ow, max_seqs=8, **kw)
    assert m.split8 == wide.split8 == 768 and m.max_rows == 32 and wide.max_rows == 64
    # so that a context of two splits does not fit at once: a workspace of eight rows of them
    m.part8 = m.part8[:K.part_floats(8, cfg.n_heads, cfg.head_dim, 1536, 768)]
    torch.manual_seed(6)
    ids = torch.randint(0, cfg.vocab, (1010,))
    for x in (m, wide):
        x.new_seq(0)
    for lo, hi in ((0, 63), (63, 900), (900, 963), (963, 1010)):
        for x in (m, wide):
            torch.cuda.synchronize()
            torch.cuda.reset_peak_memory_stats()
            before = torch.cuda.memory_allocated()
            _, x.lg = x.prefill(0, ids[lo:hi], want_logits=True)
            x.took = torch.cuda.max_memory_allocated() - before
        assert torch.equal(m.lg, wide.lg)
        if hi - lo <= 63:
            # the whole table's splits for these rows would be as large as this
            table = 4 * K.part_floats(hi - lo, cfg.n_heads, cfg.head_dim, 131072, 768)
            assert m.took < table / 2 and wide.took < table / 2, (m.took, wide.took, table)
    assert m.device_status() == 0 and wide.device_status() == 0


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("q_heads,kv_heads", [(16, 8), (32, 4)])
def test_chunks_of_heads_of_128_are_the_attention_over_their_pages(fmt, q_heads, kv_heads):
    """Two layers with heads of 128, chunks of 128 rows and a last one of 93 that ends inside a page: what the model's prefill attention
    returns for every chunk and layer is, within the roundings of the prefill kernel, the 64-bit attention over the pages that it has just
    written; and the logits are those of a model that takes 48 rows at a time, straight over the 8-bit pages."""
    import dataclasses
    from tests.kv8_reference import attend, seen_keys, values
    cfg = dataclasses.replace(C.scaled(C.drafter_0p6b(), 2), n_heads=q_heads, n_kv_heads=kv_heads)
    hq, hkv, hd = cfg.n_heads, cfg.n_kv_heads, cfg.head_dim
    kw = dict(max_seqs=2, max_ctx=1024, bf16_linears=True, kv_cache=fmt)
    m = DenseModel.random_init(cfg, seed=3, prefill_chunk=128, **kw)
    seen = []
    real = m._prefill_attend8

    def spy(li, qkv, q, seq, pos0, pos, seqv):
        out = real(li, qkv, q, seq, pos0, pos, seqv)
        pages = m.block_table[seq, :(pos0 + q.shape[0] + 15) // 16].long()
        seen.append((pos0, q.cpu(), out.clone().cpu(), m.kv[li][pages].cpu()))
        return out
    m._prefill_attend8 = spy
    torch.manual_seed(4)
    other, prompt = torch.randint(0, cfg.vocab, (200,)), torch.randint(0, cfg.vocab, (349,))
    m.new_seq(0); m.new_seq(1)
    m.prefill(0, other)
    m._stage.fill_(float("nan"))                              # whatever the staging pages held: only what is written now counts
    seen.clear()
    _, lg = m.prefill(1, prompt, want_logits=True)
    assert [s[0] for s in seen] == [0, 0, 128, 128, 256, 256] and seen[-1][1].shape[0] == 93
    for pos0, q, out, pages in seen:
        T = q.shape[0]
        k, v = (x.transpose(1, 2).reshape(-1, hkv, hd) for x in values(pages, hd, fmt))
        for t in (0, 1, 62, T - 1):
            ref, tol = attend(q[t].view(hq, hd), k, v, seen_keys(k.shape[0], pos0 + t), hq, hkv)
            # K, V and weights in bf16: 2^-8 of each, K's through the scores
            kk, vv = k[:pos0 + t + 1].abs(), v[:pos0 + t + 1].abs()
            big = (q[t].double().view(hkv, -1, hd).abs() @ kk.permute(1, 2, 0)).amax() / hd ** 0.5
            tol = tol + (3 + float(big)) * 2.0 ** -8 * vv.amax()
            off = (out[t].view(hq, hd).double() - ref).abs()
            assert bool((off <= tol).all()), (pos0, t, float((off / tol).max()))
            # and nearer than that on the whole: the roundings are independent, 2^-8 of the result's size and as much of its scores'
            assert float(off.norm()) <= 0.03 * float(ref.norm()), (pos0, t, float(off.norm() / ref.norm()))
    small = DenseModel.random_init(cfg, seed=3, prefill_chunk=48, **kw)
    small.new_seq(0)
    _, ls = small.prefill(0, prompt, want_logits=True)
    # the two differ by the roundings above in the attention of two layers, and by what these move in later bf16 roundings
    assert float((lg - ls).norm()) < 0.03 * float(ls.norm())
    assert m.device_status() == 0 and small.device_status() == 0
