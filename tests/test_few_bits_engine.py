"""Engines whose products are in 8 bits and whose cache is in 4, whole: on the host with the plain ops, on the GPU against those."""

import numpy as np
import pytest
import torch

import traces
from plain import ops_ref as R
from qwen3_runtime_amd.ops import Int8Weight
from test_cache4_gpu import codes_of, element_places

PAGES = {"tiny_a": 16, "tiny_b": 8}
GPU = pytest.mark.gpu


class FewBitOps(R.TorchOps):
    """The plain ops with weights in 8 bits and a cache in 4, by their definitions."""

    @staticmethod
    def _product(x, w):
        most = x.float().abs().amax(-1)
        top = torch.full_like(most, 127)
        q = (x.float() * torch.where(most < 2.0 ** -100, 0.0, top / most)[:, None]).round()
        sums = q.double() @ w.values[:, : w.shape[1]].double().t()
        return (sums * (most / top).double()[:, None] * w.scale.double()).float()

    def linear(self, x, w, out_f32=False):
        if not isinstance(w, Int8Weight):
            return super().linear(x, w, out_f32)
        y = self._product(x, w)
        return y if out_f32 else y.to(x.dtype)

    def linear_for_residual(self, x, w):
        return self._product(x, w) if isinstance(w, Int8Weight) else super().linear_for_residual(x, w)

    def gated_linear(self, x, w, activation="swiglu", limit=0.0, row_scale=None):
        if not isinstance(w, Int8Weight):
            return super().gated_linear(x, w, activation, limit, row_scale)
        g, u = self._product(x, w).chunk(2, -1)
        return (g * torch.sigmoid(g) * u).to(x.dtype)

    def kv_store(self, k, v, cache):
        if cache.spec.bits != 4:
            return super().kv_store(k, v, cache)
        d, ps = k.shape[-1], cache.group.page_size
        key, value = element_places(d)
        slots = cache.group.slots.long()
        page, off = slots // ps, slots % ps
        kc, kl, ks = codes_of(k)
        vc, vl, vs = codes_of(v)
        kb, vb = (torch.zeros(*k.shape[:2], d // 2, dtype=torch.uint8) for _ in range(2))
        for e in range(d):
            kb[..., key[e][0]] |= kc[..., e] << key[e][1]
            vb[..., value[e][0]] |= vc[..., e] << value[e][1]
        cache.k[page, :, off] = kb
        cache.v.view(cache.v.shape[0], -1, ps // 4, d // 2, 4)[page, :, off // 4, :, off % 4] = vb
        cache.pages["steps"][page, :, off] = torch.stack([kl, ks, vl, vs], -1)

    def qk_norm_rope_store(self, qkv, nq, nkv, d, q_w, k_w, eps, inv_freq, positions, cache, **more):
        if cache is None or cache.spec.bits != 4:
            return super().qk_norm_rope_store(qkv, nq, nkv, d, q_w, k_w, eps, inv_freq, positions, cache, **more)
        t = qkv.shape[0]
        k = torch.zeros(t, nkv, 1, d, dtype=qkv.dtype)
        v = torch.zeros(t, nkv, d, 1, dtype=qkv.dtype)
        q = R.qk_norm_rope_store(qkv, nq, nkv, d, q_w, k_w, eps, inv_freq, positions, k, v, torch.arange(t, dtype=torch.int32), 1, self.compute)
        self.kv_store(k[:, :, 0], v[..., 0], cache)
        return q

    def paged_attention(self, q, cache, ctx, nq, nkv, d, scale, window, **more):
        if cache.spec.bits != 4:
            return super().paged_attention(q, cache, ctx, nq, nkv, d, scale, window, **more)
        key, value = element_places(d)
        ps, pages = cache.group.page_size, cache.k.shape[0]
        st = cache.pages["steps"].float()
        k = torch.stack([cache.k[..., b] >> s & 15 for b, s in key], -1).float()
        fours = cache.v.view(pages, nkv, ps // 4, d // 2, 4)
        v = torch.stack([fours[..., b, :] >> s & 15 for b, s in value], -1).reshape(pages, nkv, ps, d).float()
        return R.paged_attention(q, st[..., 0:1] + st[..., 1:2] * k, (st[..., 2:3] + st[..., 3:4] * v).transpose(2, 3), ctx.cu_q, ctx.kv_lens,
                                 cache.group.block_table, ps, nq, nkv, d, scale, window, self.compute, **more)


def loaded(folder, page, pages, dtype, device, weights="model", cache_bits=None, hip_graph=False):
    from qwen3_runtime_amd.config.engine import EngineConfig
    from qwen3_runtime_amd.engine.factory import load

    cfg = EngineConfig(page_size=page, num_pages=pages, max_num_seqs=4, dtype=dtype, device=device, hip_graph=hip_graph, weights=weights, cache_bits=cache_bits)
    return load(folder, cfg, ops=FewBitOps() if device == "cpu" else None)


def logits(folder, steps, page, pages, **how):
    return traces.replay(loaded(folder, page, pages, **how), steps)


WAYS = [dict(weights="int8"), dict(cache_bits=4), dict(weights="int8", cache_bits=4)]


@pytest.fixture(scope="module")
def work(model_folders, tiny_configs):
    """tiny_b: heads of 32, which a cache of 4 bits takes."""
    cfg, page = tiny_configs["tiny_b"]
    reqs = traces.make_requests(cfg.vocab_size, [3, 17, 40, 64, 95], seed=5)
    return model_folders["tiny_b"], page, reqs


def far(got, want):
    """(median, largest) difference over the logits' deviation."""
    assert got.keys() == want.keys()
    d = np.concatenate([np.abs(np.asarray(got[k]) - np.asarray(want[k])).ravel() for k in want])
    return float(np.median(d)) / np.std([np.asarray(x) for x in want.values()]), float(d.max()) / np.std([np.asarray(x) for x in want.values()])


@pytest.mark.parametrize("way", range(3))
def test_a_host_engine_in_few_bits_is_near_the_whole_one_and_cut_does_not_matter(work, way):
    folder, page, reqs = work
    whole = logits(folder, traces.whole(reqs), page, 64, dtype="float32", device="cpu")
    few = logits(folder, traces.whole(reqs), page, 64, dtype="float32", device="cpu", **WAYS[way])
    # steps of 1 / 254 of a row's largest element in 8 bits, of 1 / 30 of a head's range in 4: per cent, and a few of ten
    assert 1e-4 < far(few, whole)[0] < 0.2
    cut = logits(folder, traces.portions(reqs), page, 64, dtype="float32", device="cpu", **WAYS[way])
    assert far(cut, few)[0] < 1e-4


@GPU
@pytest.mark.parametrize("way", range(3))
@pytest.mark.parametrize("cut", ["whole", "tail_one_by_one", "portions", "mixed"])
@pytest.mark.parametrize("graph", [False, True])
def test_the_gpu_engine_is_the_host_one(work, way, cut, graph):
    """float32 on both sides. Their sums differ in the last places, so now and then an element lies on the other side of a border between two codes,
    which is a step of 1 / 127 of a row's largest element or of 1 / 15 of a head's range in one element of one token: the median shows the sums, the
    largest difference such steps."""
    folder, page, reqs = work
    want = logits(folder, traces.whole(reqs), page, 64, dtype="float32", device="cpu", **WAYS[way])
    got = logits(folder, getattr(traces, cut)(reqs), page, 64, dtype="float32", device="cuda:0", hip_graph=graph, **WAYS[way])
    middle, most = far(got, want)
    assert middle < 1e-4 and most < 0.2, (middle, most)


@GPU
@pytest.mark.parametrize("way", range(3))
def test_the_gpu_engine_in_bfloat16(work, way):
    """What bfloat16 makes of an element of a key or value of deviation 1 is off by d = 0.015 (the bound that the repository's
    bfloat16 engines keep of their logits), so of codes a step s = 4.1 / 15 apart (the range of 32 normal elements over 15) a share of
    0.8 d / s = 0.044 falls on the other side of a border, by a whole step: sqrt(0.044) s = 0.057 of noise an element, where the
    codes themselves have s / sqrt(12) = 0.079. In 8 bits a step is 1 / 127 of a row's largest element and the same sum gives less. So
    the noise against the host's engine in few bits is at most what the few bits themselves make, beside bfloat16's own."""
    folder, page, reqs = work
    whole = logits(folder, traces.whole(reqs), page, 64, dtype="float32", device="cpu")
    want = logits(folder, traces.whole(reqs), page, 64, dtype="float32", device="cpu", **WAYS[way])
    got = logits(folder, traces.mixed(reqs), page, 64, dtype="bfloat16", device="cuda:0", hip_graph=True, **WAYS[way])
    (middle, most), (middle_of_bits, most_of_bits) = far(got, want), far(want, whole)
    assert middle < middle_of_bits + 0.015 and most < most_of_bits + 0.08, (middle, most, middle_of_bits, most_of_bits)


@GPU
def test_llm_in_few_bits():
    from qwen3_runtime_amd import LLM, SamplingParams

    prompts = [[5, 17, 3], [9, 9, 1, 250, 7]]
    for dtype in ("float32", "bfloat16"):
        llm = LLM(config="tiny_b", dtype=dtype, block_size=8, weights="int8", cache_bits=4)
        together = llm.generate(prompts, SamplingParams(temperature=0.0), max_tokens=12)
        assert [len(x) for x in together] == [12, 12]
        assert [llm.generate(p, SamplingParams(temperature=0.0), max_tokens=12) for p in prompts] == together


# ---- needs no GPU


def test_what_is_held_in_few_bits(work):
    folder, page, _ = work
    m = loaded(folder, page, 8, "float32", "cpu", weights="int8", cache_bits=4)
    whole = loaded(folder, page, 8, "float32", "cpu")
    block = m.model.blocks[0]
    assert isinstance(block.mixer.qkv, Int8Weight) and isinstance(block.mixer.o, Int8Weight) and isinstance(block.feed_forward.gate_up, Int8Weight)
    assert not isinstance(m.model.head.weight, Int8Weight)
    assert m.weight_bytes < 0.6 * whole.weight_bytes
    assert m.cache.bytes_read([100]) == 100 * 3 * 2 * 40 and whole.cache.bytes_read([100]) == 100 * 3 * 2 * 256
    a, b = (x.model.step_cost([(1, 10)], 1, 4) for x in (m, whole))
    assert a.flop == b.flop and a.total_weight_bytes < b.total_weight_bytes
    name = "model.layers.0.mlp.down_proj.weight"
    assert a.weight_bytes[name] == 96 * 272 + 4 * 96 and b.weight_bytes[name] == 96 * 272 * 4


def test_models_and_options_that_have_no_such_form_are_refused(model_folders):
    from qwen3_runtime_amd.config.engine import EngineConfig
    from qwen3_runtime_amd.engine.factory import build_model
    from qwen3_runtime_amd.registry import preset_config

    for bad in (dict(weights="int4"), dict(cache_bits=8), dict(cache_bits=2)):
        with pytest.raises(ValueError):
            EngineConfig(**bad)
    with pytest.raises(ValueError, match="heads of 32"):
        build_model(preset_config("tiny_a"), cache_bits=4)  # heads of 16
    refused = 0
    for name in ("deginex_tiny_a", "roserax_tiny_a", "zuvasun_tiny_a", "zisedra_tiny_a", "sarudra_tiny_a", "dekinex_tiny_a"):
        try:
            build_model(preset_config(name), cache_bits=4)
        except ValueError:
            refused += 1
    assert refused >= 3  # gates, latents, turned values, values of another size


def test_a_weight_that_is_not_finite_is_named(tmp_path, model_folders):
    import json
    import shutil

    from safetensors.torch import load_file, save_file

    shutil.copytree(model_folders["tiny_b"], tmp_path / "m")
    tensors = load_file(tmp_path / "m" / "model.safetensors")
    tensors["model.layers.1.mlp.down_proj.weight"][3, 5] = float("inf")
    save_file(tensors, tmp_path / "m" / "model.safetensors")
    assert json.loads((tmp_path / "m" / "config.json").read_text())
    with pytest.raises(ValueError, match="model.layers.1.mlp.down_proj"):
        loaded(tmp_path / "m", 8, 8, "float32", "cpu", weights="int8")
