"""Weights in 8 bits in every arrangement of a layer, the cache in 4 bits behind convolutions, and which models refuse it: engines over
the designs' tiny configurations, on the host with the plain ops, on the GPU against those."""

import copy

import numpy as np
import pytest
import torch

import traces
from plain import ops_ref as R
from test_few_bits_engine import FewBitOps, far
from qwen3_runtime_amd.ops import Int8Weight
from qwen3_runtime_amd.registry import preset_config, preset_names, preset_page_size

GPU = pytest.mark.gpu

# the block of a layer, and what is special about its parts
DESIGNS = {
    "deginex_tiny_a": "several streams; a q/k norm over the whole projection, clamped gates",
    "zisedra_tiny_a": "two mixers side by side, one with values of another size",
    "roserax_tiny_a": "norms on both sides; a feed-forward without a gate",
    "zuvasun_tiny_a": "mixer and feed-forward side by side in one scaled sum",
    "sarudra_tiny_a": "norms behind the sub-layers, in groups; turned values",
    "dekinex_tiny_a": "one scaled sum, a span of layers run twice; convolutions, rows in another order",
    "tiny_b": "a norm in front of each sub-layer",
}


class Ops(FewBitOps):
    """... with the gate's other activations."""

    def gated_linear(self, x, w, activation="swiglu", limit=0.0, row_scale=None):
        if not isinstance(w, Int8Weight):
            return super().gated_linear(x, w, activation, limit, row_scale)
        gate, up = self._product(x, w).chunk(2, -1)
        return R.gated(gate, up, activation, limit).to(x.dtype)


def behind_convolutions():
    """dekinex_tiny_a with heads of 32 and 64 whose values are as wide."""
    raw = copy.deepcopy(preset_config("dekinex_tiny_a"))
    for i, dim in ((1, 32), (3, 64)):
        raw["layers"][i]["mixer"].update(dim=dim, vdim=dim)
    return raw


@pytest.fixture(scope="module")
def folders(tmp_path_factory):
    from qwen3_runtime_amd.weights import write_model_folder

    made = {}

    def get(name):
        if name not in made:
            raw = behind_convolutions() if name == "behind convolutions" else preset_config(name)
            made[name] = tmp_path_factory.mktemp("designs") / name.replace(" ", "_")
            made[name].mkdir()
            write_model_folder(made[name], raw, seed=5)
        return made[name]

    return get


def logits(folder, page, cut, dtype="float32", device="cpu", hip_graph=False, **bits):
    from qwen3_runtime_amd.config.engine import EngineConfig
    from qwen3_runtime_amd.engine.factory import load

    cfg = EngineConfig(page_size=page, num_pages=128, max_num_seqs=4, dtype=dtype, device=device, hip_graph=hip_graph, **bits)
    m = load(folder, cfg, ops=Ops() if device == "cpu" else None)
    return traces.replay(m, cut(traces.make_requests(m.runner.vocab_size, [3, 17, 40, 95], seed=5)))


def rows_off(got, want):
    """Of every row its largest difference over the logits' deviation."""
    spread = np.std([np.asarray(x) for x in want.values()])
    return np.array([np.abs(np.asarray(got[k]) - np.asarray(want[k])).max() for k in want]) / spread


CASES = [(name, dict(weights="int8")) for name in DESIGNS] + [("behind convolutions", dict(cache_bits=4)), ("behind convolutions", dict(weights="int8", cache_bits=4))]
IDS = [f"{name}-{'-'.join(map(str, bits.values()))}".replace(" ", "_") for name, bits in CASES]


def page_of(name):
    return preset_page_size("dekinex_tiny_a" if name == "behind convolutions" else name)


@pytest.mark.parametrize("name,bits", CASES, ids=IDS)
def test_a_host_engine_of_every_design(folders, name, bits):
    """Near the whole engine: a row's codes are 1 / 254 of its largest element off, a head's a thirtieth of its range; and the same however
    the requests are cut, but for an element now and then that lies on the other side of a border, or a token that goes to another expert."""
    whole = logits(folders(name), page_of(name), traces.whole)
    few = logits(folders(name), page_of(name), traces.whole, **bits)
    assert 1e-4 < far(few, whole)[0] < 0.2
    cut = logits(folders(name), page_of(name), traces.portions, **bits)
    assert far(cut, few)[0] < 1e-4 and np.quantile(rows_off(cut, few), 0.9) < 0.05


@pytest.fixture
def planes(monkeypatch):
    """Products for the residual of more than 32 rows in two planes (halves, whose sum has the same bits), as they come by K of 2,048 and
    more: what reads them has to take planes in every design."""
    from qwen3_runtime_amd.ops.hip import HipOps

    whole, made = HipOps.linear_for_residual, []

    def halves(self, x, w):
        y = whole(self, x, w)
        if isinstance(w, Int8Weight) and self.residual_planes and x.shape[0] > 32 and y.dim() == 2:
            made.append(w.shape)
            y = torch.stack([y / 2, y / 2])
        return y

    monkeypatch.setattr(HipOps, "linear_for_residual", halves)
    return made


@GPU
@pytest.mark.parametrize("name,bits", CASES, ids=IDS)
def test_the_gpu_engine_of_every_design_is_the_host_one(folders, planes, name, bits):
    """float32 on both sides, steps of more than 32 rows among them. The median shows the sums; a code on the other side of its border moves what
    follows of its request by some hundredths (0.02 where the host's own steps are cut otherwise), and that falls on few rows."""
    want = logits(folders(name), page_of(name), traces.whole, **bits)
    got = logits(folders(name), page_of(name), traces.whole, device="cuda:0", **bits)
    off = rows_off(got, want)
    assert far(got, want)[0] < 1e-4 and np.quantile(off, 0.9) < 0.05, (far(got, want), np.quantile(off, [0.5, 0.9, 1.0]))
    assert planes or "weights" not in bits


@GPU
@pytest.mark.parametrize("cut", ["whole", "mixed"])
@pytest.mark.parametrize("name,bits", CASES, ids=IDS)
def test_the_gpu_engine_of_every_design_in_bfloat16(folders, planes, name, bits, cut):
    """The noise of codes that bfloat16's roundings bring to the other side of a border is at most that of the codes themselves, beside bfloat16's
    own (a root mean square of 0.015 of the logits' deviation, which the median is under)."""
    whole = logits(folders(name), page_of(name), traces.whole)
    want = logits(folders(name), page_of(name), traces.whole, **bits)
    got = logits(folders(name), page_of(name), getattr(traces, cut), dtype="bfloat16", device="cuda:0", hip_graph=True, **bits)
    assert far(got, want)[0] < far(want, whole)[0] + 0.015, (far(got, want), far(want, whole))


# ---- needs no GPU

TAKEN = {"tiny_b", "qwen3_4b", "qwen3_8b", "qwen3_32b", "dekinex_2b", "dekinex_4b", "dekinex_8b"}
REFUSED = {
    "heads of 32 to 256": {"tiny_a", "deginex_tiny_b", "zisedra_tiny_a", "zisedra_tiny_b", "roserax_tiny_a", "roserax_tiny_b", "roserax_2b", "roserax_4b",
                           "roserax_8b", "zuvasun_tiny_a", "zuvasun_tiny_b", "zuvasun_2b", "zuvasun_4b", "zuvasun_8b", "sarudra_tiny_a", "sarudra_tiny_b",
                           "dekinex_tiny_a", "dekinex_tiny_b"},
    "goes without": {"deginex_tiny_a", "deginex_4b", "deginex_4b_moe", "deginex_8b_moe", "sarudra_2b", "sarudra_4b", "sarudra_8b"},
    "'side_by_side' does not read": {"zisedra_2b", "zisedra_4b", "zisedra_8b"},
}


def test_which_models_take_a_cache_of_4_bits():
    from qwen3_runtime_amd.engine.factory import build_model

    reasons = {name: why for why, names in REFUSED.items() for name in names}
    for name in TAKEN:
        model = build_model(preset_config(name), cache_bits=4)[1]
        assert {s.bits for s in model.plan.caches if s.paged} == {4}
    for name, why in reasons.items():
        with pytest.raises(ValueError, match=why):
            build_model(preset_config(name), cache_bits=4)
    assert {n for n in preset_names() if n.split("_")[0] in ("tiny", "qwen3", "deginex", "zisedra", "roserax", "zuvasun", "sarudra", "dekinex")} == TAKEN | set(reasons)
