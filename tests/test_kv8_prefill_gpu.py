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
