"""The serving engine with the paged 8-bit cache and the 4-bit weights."""

import pytest
import torch

from marin_experiments_b200.data.tokenize import ByteTokenizer
from marin_experiments_b200.models.qwen3 import Qwen3Config, Qwen3Model
from marin_experiments_b200.ops import api
from marin_experiments_b200.serving.engine import Engine, SamplingParams

pytestmark = pytest.mark.gpu


def rel(a, b):
    return ((a.float() - b.float()).norm() / b.float().norm().clamp_min(1e-12)).item()


def config(hd=64, heads=4, kv=2, **kw):
    return Qwen3Config(vocab_size=512, hidden_dim=256, intermediate_dim=256, num_layers=2, num_heads=heads,
                       num_kv_heads=kv, head_dim=hd, rope_theta=10000.0, max_seq_len=512, **kw)


def round_weights(model, group):
    """The model with the weights that 4 bits hold (exact in fp32)."""
    with torch.no_grad():
        for p in [w for L in model.layers for w in (L.w_q, L.w_k, L.w_v, L.w_o, L.w_gate_up, L.w_down)] + [model.lm_head]:
            p.copy_(api.dequantize_w4(*api.quantize_w4(p.to(torch.bfloat16), group)))


@pytest.mark.parametrize("kv_cache,weights,hd,heads,kv,graphs", [("fp8", "bf16", 64, 4, 2, True), ("bf16", "int4", 128, 2, 2, True),
                                                                 ("fp8", "int4", 128, 4, 1, True), ("fp8", "int4", 64, 4, 4, False)])
def test_prefill_and_decode_match_reference(kv_cache, weights, hd, heads, kv, graphs):
    """Against the fp32 model (with the rounded weights). An e4m3 cache is off by 2^-4 of a value at
    most, 2^-4 / sqrt(3) = 0.036 in the mean square; half of a layer's output passes through it, so
    the logits stay within 0.06."""
    cfg = config(hd, heads, kv)
    ref = Qwen3Model(cfg).init_weights(3)
    gpu = Qwen3Model(cfg)
    gpu.load_state_dict(ref.state_dict())
    gpu = gpu.cuda()
    eng = Engine(gpu, ByteTokenizer(), max_batch=2, max_len=512, use_graphs=graphs, kv_cache=kv_cache, weights=weights,
                 page_size=32, group=64)
    if weights == "int4":
        round_weights(ref, 64)
    g = torch.Generator().manual_seed(0)
    seqs = [torch.randint(0, 512, (n,), generator=g).tolist() for n in (90, 31)]  # above and below 64 rows
    for slot, s in enumerate(seqs):
        assert rel(eng._prefill(s, slot).cpu(), ref.forward_reference(torch.tensor([s]))[:, -1]) < 4e-2
    pos = torch.tensor([len(s) for s in seqs], dtype=torch.int32, device="cuda")
    bound = 6e-2 if kv_cache == "fp8" else 4e-2
    for step in range(5):  # the second sequence passes a page end
        nxt = torch.randint(0, 512, (2,), generator=g)
        out = eng._decode(nxt.cuda(), pos)
        for j in range(2):
            seqs[j].append(int(nxt[j]))
            want = ref.forward_reference(torch.tensor([seqs[j]]))[:, -1]
            assert rel(out[j:j + 1].cpu(), want) < bound, (step, j)
        pos = pos + 1
    if kv_cache == "fp8":
        assert eng.lens.tolist() == [len(s) for s in seqs]
        assert int(eng.free_count) == eng.pages - sum(-(-len(s) // 32) for s in seqs)


def test_pages_are_given_back_between_batches():
    """A pool of far fewer pages than full-length sequences need serves batch after batch; graphs and
    eager steps give the same tokens; a prompt set that cannot fit is refused."""
    m = Qwen3Model(config()).init_weights(5).cuda()
    tok = ByteTokenizer()
    engines = [Engine(m, tok, max_batch=3, max_len=512, kv_cache="fp8", weights="int4", page_size=32, pages=9,
                      use_graphs=g) for g in (True, False)]
    p = SamplingParams(max_tokens=40, temperature=0.0)
    prompts = [tok.encode(t) for t in ("alpha", "beta gamma delta", "a" * 50, "x", "yy" * 20, "last one")]
    a, b = (e.generate_ids(prompts, p) for e in engines)
    assert a == b and a == engines[0].generate_ids(prompts, p)
    for e in engines:
        assert int(e.free_count) + sum(-(-n // 32) for n in e.lens.tolist()) == 9
        used = e.free_pages[: int(e.free_count)].tolist() + [x for x in e.tables.flatten().tolist() if x >= 0]
        assert sorted(used) == list(range(9))  # every page is free or in one table
        with pytest.raises(ValueError):
            e.generate_ids([[1] * 300], p)


def test_refresh_weights_in_place():
    """Captured graphs keep sampling, now from the new weights, like a fresh engine."""
    m = Qwen3Model(config()).init_weights(5).cuda()
    tok = ByteTokenizer()
    kw = dict(max_batch=2, max_len=256, kv_cache="fp8", weights="int4")
    eng = Engine(m, tok, **kw)
    p = SamplingParams(max_tokens=10, temperature=0.0)
    prompts = [tok.encode("alpha"), tok.encode("beta gamma")]
    first = eng.generate_ids(prompts, p)
    with torch.no_grad():
        for L in m.layers:
            L.w_o.mul_(-1.5)
            L.w_down.add_(0.05 * torch.randn_like(L.w_down))
        m.embed.mul_(1.3)
        m.lm_head.mul_(-1)
    eng.refresh_weights()
    again = eng.generate_ids(prompts, p)
    assert again == Engine(m, tok, **kw).generate_ids(prompts, p) and again != first


def test_options_that_the_engine_refuses():
    m = Qwen3Model(config()).init_weights(5).cuda()
    for kw in ({"kv_cache": "int8"}, {"weights": "fp4"}, {"kv_cache": "fp8", "page_size": 48},
               {"weights": "int4", "group": 16}, {"kv_cache": "fp8", "pages": 0}):
        with pytest.raises(ValueError):
            Engine(m, ByteTokenizer(), max_batch=2, max_len=64, **kw)
