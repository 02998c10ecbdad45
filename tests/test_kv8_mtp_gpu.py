"""The multi-token-prediction head over 8-bit pages drafts, and what is decoded with it is what is decoded without."""
import pytest
import torch

from agens_engine_b200.models import config as C
from agens_engine_b200.models import oracle as O
from agens_engine_b200.models.dense import DenseModel
from agens_engine_b200.models.mtp import MtpHead
from agens_engine_b200.ops import kv8 as K
from agens_engine_b200.spec import MtpSource, SpecDecoder

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("target,head", [("int8", None), ("fp8", None), ("int8", "bf16"), ("bf16", "fp8")])
def test_mtp_head_with_8_bit_pages(target, head):
    cfg = C.oracle_tiny()
    ow = O.random_weights(cfg, seed=0)
    torch.manual_seed(11)
    prompt = torch.randint(0, cfg.vocab, (77,)).tolist()              # chunks of 32, 32 and a 13-row tail
    kw = dict(max_seqs=2, max_ctx=512, prefill_chunk=32, kv_cache=target)
    one = DenseModel.from_oracle(ow, **kw)
    plain = SpecDecoder(one, [], max_drafts=0).generate(0, prompt, 24, None)
    m = DenseModel.from_oracle(ow, **kw)
    h = MtpHead.random_init_for(m, **({} if head is None else {"kv_cache": head}))
    fmt = head or target
    assert h.cfg.kv_cache == fmt and h.kv8 == (None if fmt == "bf16" else fmt) and (head is not None or h.split8 == m.split8)
    dec = SpecDecoder(m, [MtpSource(h, depth=2)], max_drafts=4)
    out = [dec.begin(0, prompt)]
    assert h.seq_len_host[0] == len(prompt)                            # an entry for every position of the prompt
    if h.kv8:
        first = K.kv_read8(h.kv[0], h.kv8, h.block_table[0, :5], n_tokens=77)
        assert bool((first.float().abs().amax(-1).transpose(1, 2).reshape(5, cfg.n_kv_heads, -1)[:4] > 0).all())
    while len(out) < 24:
        out += dec.step([0])[0]
    assert out[:24] == plain and dec.stats.by_source.get("mtp", [0, 0])[0] > 0
    assert m.device_status() == 0 and h.device_status() == 0


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
def test_the_head_drafts_as_over_bf16_pages(fmt):
    """The same hidden rows and tokens through heads over bf16 and 8-bit pages: the layer's output differs by what 8 bits of K and V
    make (int8 a 1 / 254 of a row's largest value at most, a third of that rms, e4m3 2^-4 at most, 2.5 % rms), attention being one of the
    output's two parts: 3 % (10 %) of its norm leave room."""
    cfg = C.oracle_tiny()
    m = DenseModel.from_oracle(O.random_weights(cfg, seed=0), max_seqs=2, max_ctx=512)
    a, b = (MtpHead.random_init_for(m, kv_cache=f) for f in ("bf16", fmt))
    torch.manual_seed(3)
    n = 60
    toks = torch.randint(0, cfg.vocab, (n,))
    hidden = torch.randn(n, cfg.d_model, device=m.dev).to(torch.bfloat16)
    outs = []
    for h in (a, b):
        h.new_seq(0)
        h.prefill_pairs(0, toks[:52], hidden[:52])
        h.forward_mtp(toks[52:].tolist(), hidden[52:], [0] * 8)
        outs.append(h.h_a[:8].float().clone())
    assert float((outs[0] - outs[1]).norm()) < (0.03 if fmt == "int8" else 0.10) * float(outs[0].norm())
    assert not torch.equal(outs[0], outs[1]) and b.device_status() == 0
