"""A model served from a paged cache against the same model on its contiguous caches, sequence by sequence."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
if torch.cuda.is_available():
    from mojolearn_b200 import lowbit
    from mojolearn_b200.models import CausalLM, CausalLMConfig, PagedLM


def model(seed=0, weight=None, **kw):
    cfg = CausalLMConfig(vocab=512, d_model=256, n_layers=3, **dict({"n_heads": 8, "n_kv_heads": 2, "head_dim": 64, "intermediate": 512, "max_positions": 1024}, **kw))
    r = np.random.default_rng(seed)
    w = {"model.embed_tokens.weight": r.standard_normal((512, 256)) * 0.5, "model.norm.weight": 1 + 0.1 * r.standard_normal(256), "lm_head.weight": r.standard_normal((512, 256)) * 0.1}
    if cfg.positions == "learned":
        w["model.embed_positions.weight"] = r.standard_normal((1024, 256)) * 0.1
    hd = cfg.head_dim
    for i in range(3):
        p = "model.layers.%d." % i
        for n in ("input_layernorm", "post_attention_layernorm"):
            w[p + n + ".weight"] = 1 + 0.1 * r.standard_normal(256)
        for n, rows, cols in (("self_attn.q_proj", 8 * hd, 256), ("self_attn.k_proj", cfg.n_kv_heads * hd, 256), ("self_attn.v_proj", cfg.n_kv_heads * hd, 256),
                              ("self_attn.o_proj", 256, 8 * hd), ("mlp.gate_proj", 512, 256), ("mlp.up_proj", 512, 256), ("mlp.down_proj", 256, 512)):
            w[p + n + ".weight"] = r.standard_normal((rows, cols)) * 0.06
        if cfg.qk_norm:
            for n in ("q_norm", "k_norm"):
                w[p + "self_attn." + n + ".weight"] = 1 + 0.1 * r.standard_normal(hd)
    w = {k: np.asarray(v, dtype=np.float32) for k, v in w.items()}
    if weight:
        w = {k: lowbit.pack_one(v, weight) if "_proj" in k else v for k, v in w.items()}
    return CausalLM(cfg, w)


@pytest.mark.parametrize("options", [{}, {"window": 40}, {"qk_norm": True}, {"attn_softcap": 20.0}, {"rope_dim": 32}, {"positions": "learned"}, {"n_kv_heads": 8, "head_dim": 32},
                                     {"weight": "int8"}])
@pytest.mark.parametrize("cache", ["float32", "bfloat16"])
def test_logits_of_ragged_chunks(options, cache):
    """Prompts of several lengths in chunks, with single tokens of others beside them. float32 pages: the logits differ from the contiguous
    model's by rounding (three blocks, each about 1e-6 of its size); bfloat16 ones by what 8 bits of keys and values leave (2^-9 each)."""
    lm = model(**options)
    served = PagedLM(lm, 64, page=16, cache=cache)
    r = np.random.default_rng(1)
    ids = [r.integers(0, 512, n).astype(np.int32) for n in (70, 3, 129, 1)]
    names = [served.open() for _ in ids]
    served.feed(names[:1], [ids[0][:33]])
    served.feed([names[2], names[0]], [ids[2][:64], ids[0][33:34]])
    served.feed([names[1], names[2]], [ids[1], ids[2][64:128]])
    got = served.feed([names[0], names[3], names[2]], [ids[0][34:], ids[3], ids[2][128:]])
    lm.check_status()
    for row, x in zip(got, (ids[0], ids[3], ids[2])):
        want = torch.from_numpy(lm.forward(x[None])[0, -1]).cuda()
        off = float((row - want).norm() / want.norm())
        assert off <= (2e-5 if cache == "float32" else 2e-2), off
    assert [served.length(n) for n in names] == [70, 3, 129, 1]


def test_generate_is_the_contiguous_models():
    lm = model(seed=3)
    served = PagedLM(lm, 40, page=16, cache="float32")
    r = np.random.default_rng(2)
    prompts = [r.integers(0, 512, n).astype(np.int32) for n in (40, 5, 17)]
    for _ in range(2):  # pages come back
        got = served.generate(prompts, 12, chunk=16)
        for p, g in zip(prompts, got):
            assert g.tolist() == lm.generate(p[None], 12)[0].tolist()
    assert len(served.cache.free) == 40


def test_a_pool_that_is_too_small_refuses_and_keeps_what_it_has():
    lm = model()
    served = PagedLM(lm, 3, page=16, cache="bfloat16")
    a = served.open()
    first = served.feed([a], [np.arange(10)])
    with pytest.raises(ValueError, match="REFUSED"):
        served.feed([a], [np.arange(60)])
    assert served.length(a) == 10
    b = served.open()
    assert torch.equal(served.feed([b], [np.arange(10)]), first)
    with pytest.raises(ValueError):
        served.feed([a, b], [np.arange(3)])
    with pytest.raises(ValueError):
        served.feed([a], [np.zeros(0)])
    with pytest.raises(ValueError, match="max_positions"):
        served.feed([a], [np.zeros(2000)])
    with pytest.raises(ValueError):
        PagedLM(lm, 3, cache="int8")
