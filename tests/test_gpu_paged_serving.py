"""`PagedCache` and `PagedLM` where a call fails or is refused, and at long positions."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
if torch.cuda.is_available():
    from mojolearn_b200 import paged
    from mojolearn_b200.models import CausalLM, CausalLMConfig, PagedLM


def model(layers=3, **kw):
    cfg = CausalLMConfig(vocab=256, d_model=128, n_layers=layers, **dict({"n_heads": 4, "n_kv_heads": 2, "head_dim": 32, "intermediate": 256, "max_positions": 1024}, **kw))
    r = np.random.default_rng(5)
    hd = cfg.head_dim
    w = {"model.embed_tokens.weight": r.standard_normal((256, 128)) * 0.5, "model.norm.weight": np.ones(128), "lm_head.weight": r.standard_normal((256, 128)) * 0.1}
    for i in range(layers):
        p = "model.layers.%d." % i
        for n in ("input_layernorm", "post_attention_layernorm"):
            w[p + n + ".weight"] = np.ones(128)
        for n, rows, cols in (("self_attn.q_proj", 4 * hd, 128), ("self_attn.k_proj", 2 * hd, 128), ("self_attn.v_proj", 2 * hd, 128), ("self_attn.o_proj", 128, 4 * hd),
                              ("mlp.gate_proj", 256, 128), ("mlp.up_proj", 256, 128), ("mlp.down_proj", 128, 256)):
            w[p + n + ".weight"] = r.standard_normal((rows, cols)) * 0.08
    return CausalLM(cfg, {k: np.asarray(v, dtype=np.float32) for k, v in w.items()})


@pytest.mark.parametrize("block", [0, 1, 2])
def test_a_call_that_fails_leaves_its_sequences_as_they_were(block, monkeypatch):
    lm = model()
    served, clean = PagedLM(lm, 20, page=16), PagedLM(lm, 20, page=16)
    first, more = np.arange(10), np.arange(40) + 3
    names = []
    for s in (served, clean):
        a, b = s.open(), s.open()
        s.feed([a], [first])
        names.append((a, b))
    free, held = list(served.cache.free), list(served.cache.held[names[0][0]])

    def fail(*args, **kw):
        raise RuntimeError("out of memory, say")

    with monkeypatch.context() as m:
        m.setattr(lm.blocks[block], "forward_rows", fail)
        with pytest.raises(RuntimeError, match="say"):
            served.feed(list(names[0]), [more, first])
    assert [served.length(n) for n in names[0]] == [10, 0]
    assert sorted(served.cache.free) == sorted(free) and served.cache.held[names[0][0]] == held
    assert torch.equal(served.feed(list(names[0]), [more[:7], first]), clean.feed(list(names[1]), [more[:7], first]))


def test_tables_that_cannot_be_made_take_no_pages(monkeypatch):
    cache = paged.PagedCache(8, 2, 64, page=16)
    a = cache.open()
    cache.extend([a], [5])

    def fail(*args, **kw):
        raise RuntimeError("no pinned memory, say")

    with monkeypatch.context() as m:
        m.setattr(paged.torch, "tensor", fail)
        with pytest.raises(RuntimeError, match="say"):
            cache.extend([a], [40])
    assert cache.length[a] == 5 and len(cache.held[a]) == 1 and len(cache.free) == 7


@pytest.mark.parametrize("kw", [{"page": 24}, {"page": 8}, {"page": 512}, {"page": 0}, {"head_dim": 12}, {"head_dim": 136}, {"head_dim": 0}, {"n_kv_heads": 0}])
def test_a_pool_that_no_call_would_take_is_refused(kw):
    with pytest.raises(ValueError):
        paged.PagedCache(4, kw.pop("n_kv_heads", 2), kw.pop("head_dim", 64), **kw)


def test_a_model_whose_heads_no_call_would_take_is_refused():
    with pytest.raises(ValueError, match="head_dim"):
        PagedLM(model(layers=1, head_dim=12), 4)
    with pytest.raises(ValueError, match="page"):
        PagedLM(model(layers=1), 4, page=24)


def test_a_model_of_more_positions_than_its_rotation_has():
    """`CausalLM` takes such a model and refuses the positions past the rotation's domain; so does `PagedLM`."""
    lm = model(layers=1, max_positions=20000)
    served = PagedLM(lm, 600, page=16, cache="float32")
    a = served.open()
    ids = np.arange(30, dtype=np.int32)
    row, want = served.feed([a], [ids])[0], torch.from_numpy(lm.forward(ids[None])[0, -1]).cuda()
    assert float((row - want).norm() / want.norm()) <= 2e-5
    for n in (8192 - 30 + 1, 9000):
        with pytest.raises(ValueError, match="absolute position"):
            served.feed([a], [np.zeros(n, dtype=np.int32)])
    assert served.length(a) == 30
    served.feed([a], [np.zeros(8192 - 30, dtype=np.int32)])
    lm.check_status()
    stretched = PagedLM(model(layers=1, max_positions=20000, rope_scaling={"rope_type": "linear", "factor": 2.0}), 1200, page=16)
    b = stretched.open()
    stretched.feed([b], [np.zeros(9000, dtype=np.int32)])
    stretched.lm.check_status()
    with pytest.raises(ValueError, match="absolute position"):
        stretched.feed([b], [np.zeros(16384 - 9000 + 1, dtype=np.int32)])


def test_ids_that_are_no_integers():
    lm = model(layers=1)
    served = PagedLM(lm, 8, page=16)
    a = served.open()
    for ids in (np.array([1.5, 2.0]), [0.5], np.array([True])):
        with pytest.raises(TypeError, match="integers"):
            served.feed([a], [ids])
        with pytest.raises(TypeError, match="integers"):
            served.generate([ids], 2)
    assert served.length(a) == 0 and len(served.cache.free) == 8
    assert torch.equal(served.feed([a], [[1, 2]]), served.feed([served.open()], [np.array([1, 2], dtype=np.int64)]))
