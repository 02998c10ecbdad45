"""The dense model with an 8-bit KV cache: the same steps, sequences and sessions as with bf16 pages."""
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


def _model(ow, fmt, **kw):
    m = DenseModel.from_oracle(ow, kv_cache=fmt, **{"max_seqs": 3, "max_ctx": 512, **kw})
    assert m.kv[0].dtype == torch.uint8 and m.cfg.kv_cache == fmt
    return m


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("n", [5, 40, 150])
def test_logits_are_near_the_oracles(tiny, fmt, n):
    """Prompts that run as a small step, over 8-bit pages as they are, and over pages read back.  The bf16 model is held to 5 % of the
    largest logit; an e4m3 number is off by 2^-4 at most, 2.5 % rms, which two layers bring to 3.5 % of the logits' rms, four times
    that at the worst of a thousand, a third of which relative to the largest: 5 % more.  int8 is off by a sixth of that."""
    cfg, ow = tiny
    torch.manual_seed(n)
    prompt = torch.randint(0, cfg.vocab, (n,))
    _, ref = O.OracleModel(ow, mirror=False).generate_greedy(prompt, 1)
    m = _model(ow, fmt)
    m.new_seq(0)
    _, lg = m.prefill(0, prompt, want_logits=True)
    err = (lg.cpu() - ref[0]).abs().max().item()
    assert err < (0.06 if fmt == "int8" else 0.10) * ref[0].abs().max().item(), err
    assert m.device_status() == 0


@pytest.mark.parametrize("fmt", FMTS)
def test_rows_do_not_depend_on_their_company(tiny, fmt):
    """A verify block gives the bits of single steps, rows of several sequences those of each alone, and a replayed graph those of the
    eager step."""
    cfg, ow = tiny
    torch.manual_seed(1)
    m = _model(ow, fmt)
    p0, p1 = torch.randint(0, cfg.vocab, (140,)), torch.randint(0, cfg.vocab, (23,))
    for s, p in ((0, p0), (1, p1), (2, p0)):
        m.new_seq(s)
        m.prefill(s, p)
    cont = torch.randint(0, cfg.vocab, (6,)).tolist()
    singles = [m.forward_rows([t], [0], want_logits=True)[1][0] for t in cont]
    _, block = m.forward_rows(cont, [2] * 6, want_logits=True)
    assert all(torch.equal(a, b) for a, b in zip(block, singles))
    m.truncate(0, 140); m.truncate(2, 140)
    _, a = m.forward_rows([cont[0]], [0], want_logits=True)
    _, b = m.forward_rows([cont[1], cont[0]], [1, 2], want_logits=True)
    assert torch.equal(a[0], b[1])
    m.row_graphs = True
    m.truncate(0, 140)
    _, c = m.forward_rows([cont[0]], [0], want_logits=True)
    assert torch.equal(a[0], c[0]) and m.device_status() == 0


@pytest.mark.parametrize("fmt", FMTS)
def test_decode_graph_gives_the_eager_tokens(tiny, fmt):
    cfg, ow = tiny
    torch.manual_seed(2)
    m = _model(ow, fmt, prefill_chunk=64)
    prompt = torch.randint(0, cfg.vocab, (100,))
    m.new_seq(0)
    toks = m.generate_greedy(0, prompt, 24).tolist()
    m.new_seq(1)
    first, _ = m.prefill(1, prompt)
    eager = [first]
    for _ in range(23):
        eager.append(int(m.forward_rows([eager[-1]], [1])[0][0]))
    assert toks == eager
    bf = DenseModel.from_oracle(ow, max_seqs=1, max_ctx=512)
    assert bf.launches_per_step(1) == m.launches_per_step(1) == 2 + 7 * cfg.n_layers + 2
    assert _model(ow, fmt, max_ctx=128).launches_per_step(1) == 2 + 6 * cfg.n_layers + 2
    assert m.cfg.kv_bytes_per_token() * m.n_pages * 16 == sum(t.numel() for t in m.kv) < 0.57 * bf.cfg.kv_bytes_per_token() * m.n_pages * 16


@pytest.mark.parametrize("fmt", FMTS)
def test_fork_park_and_sessions_keep_the_bits(tiny, fmt, tmp_path):
    cfg, ow = tiny
    torch.manual_seed(3)
    m = _model(ow, fmt, max_seqs=4)
    prompt = torch.randint(0, cfg.vocab, (75,))
    m.new_seq(0)
    m.prefill(0, prompt)
    m.fork(0, 1)
    path = str(tmp_path / "s.safetensors")
    m.save_session(0, path, tokens=prompt.tolist())
    blob = m.park(0)
    assert blob["kv"].dtype == torch.uint8
    m.unpark(2, blob)
    assert m.load_session(3, path) == prompt.tolist()
    _, lg = m.forward_rows([7, 7, 7], [1, 2, 3], want_logits=True)
    assert torch.equal(lg[0], lg[1]) and torch.equal(lg[0], lg[2])
    for other in ("bf16", *(f for f in FMTS if f != fmt)):
        with pytest.raises(ValueError, match="session"):
            o = DenseModel.from_oracle(ow, max_seqs=1, max_ctx=512, kv_cache=other)
            o.load_session(0, path)


def test_the_128_wide_heads_prefill_on_the_tensor_cores():
    """Heads of 128 (the tcgen05 prefill attention over pages read back), chunk after chunk, against a model with bf16 pages that
    hold the same values: K and V of the 8-bit model, read back and put into its pool."""
    cfg = C.scaled(C.drafter_0p6b(), 1)
    kw = dict(max_seqs=1, max_ctx=640, prefill_chunk=128, bf16_linears=True)
    m = DenseModel.random_init(cfg, seed=3, kv_cache="int8", **kw)
    b = DenseModel.random_init(cfg, seed=3, **kw)
    torch.manual_seed(4)
    prompt = torch.randint(0, cfg.vocab, (300,))
    for x in (m, b):
        x.new_seq(0)
    m.prefill(0, prompt)
    b.prefill(0, prompt[:1])
    b.reserve(0, 300)
    back = K.kv_read8(m.kv[0], "int8", m.block_table[0, :19], n_tokens=300)
    b.kv[0][b.block_table[0, :19].long()] = back
    b.seq_len_host[0] = 300
    b.seq_len[0] = 300
    # the new token's attention reads the same 300 rows on both sides but for the last rounding of 8-bit values to bf16 (2^-9 rms 2^-10)
    # and its own K and V: below 1 % of the logits
    _, lm = m.forward_rows([11], [0], want_logits=True)
    _, lb = b.forward_rows([11], [0], want_logits=True)
    assert (lm - lb).norm() < 0.01 * lb.norm()
    assert m.device_status() == 0


def test_image_positions(tiny):
    """Three-axis rotary positions and image rows reach the 8-bit store."""
    cfg, ow = tiny
    m = _model(ow, "int8", prefill_chunk=64)
    torch.manual_seed(5)
    n = 90
    ids = torch.randint(0, cfg.vocab, (n,))
    pos3 = torch.arange(n, dtype=torch.int32).repeat(3, 1)
    axis = torch.arange(cfg.head_dim // 2, dtype=torch.uint8) % 3
    m.new_seq(0); m.new_seq(1)
    _, a = m.prefill(0, ids, want_logits=True)
    _, b = m.prefill(1, ids, want_logits=True, rope_pos3=pos3, pair_axis=axis, rope_next=n + 5)       # all axes alike: plain positions
    assert torch.equal(a, b)
    pos3[1, 20:50] += 3
    m.free_seq(1); m.new_seq(1)
    _, c = m.prefill(1, ids, want_logits=True, rope_pos3=pos3, pair_axis=axis, rope_next=n + 5)
    assert not torch.equal(a, c)
    m.forward_rows([3], [1])
    assert m.device_status() == 0


def test_what_an_8_bit_model_does_not_do(tiny):
    cfg, ow = tiny
    m = _model(ow, "int8")
    with pytest.raises(ValueError, match="tier"):
        m.enable_host_tier(64)
    assert not m.enable_step(True) and m.step is None
    with pytest.raises(ValueError, match="kv_cache"):
        DenseModel.from_oracle(ow, kv_cache="int4")


def test_engine_serves_with_8_bit_pages(tiny):
    """The serving loop, speculation by copy lookup included: batched requests give the tokens of single runs."""
    from agens_engine_b200.serve.engine import Engine
    from agens_engine_b200.spec import CopyLookupSource, SpecDecoder
    from tests.test_engine_gpu import Collector
    cfg, ow = tiny
    torch.manual_seed(11)
    prompts = [torch.randint(0, cfg.vocab, (n,)).tolist() for n in (5, 300, 47, 130)]
    for drafts in (0, 3):
        want = []
        for p in prompts:
            one = _model(ow, "fp8", max_seqs=1, prefill_chunk=128)
            one.set_linear_path(1 if drafts else None)       # what the engine pins for steps of more than eight rows
            want.append(SpecDecoder(one, [], max_drafts=0).generate(0, p, 24, None))
        m = _model(ow, "fp8", max_seqs=4, prefill_chunk=128)
        col = Collector()
        eng = Engine(m, col, sources_factory=(lambda: [CopyLookupSource()]) if drafts else None, max_drafts=drafts)
        rids = [eng.submit(p, {"max_new_tokens": 24}) for p in prompts]
        eng.run_until_idle(10000)
        assert eng.idle() and not col.err
        assert [col.toks[r] for r in rids] == want
        assert m.free_pages() == m.n_pages and m.device_status() == 0
