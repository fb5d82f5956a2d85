"""What products and caches in few bits promise around their kernels: workspaces, launches that follow from a step's lengths alone, what
is held. Needs no GPU but where marked."""

import weakref

import pytest
import torch

GPU = pytest.mark.gpu


def host_step(q_lens, kv_lens, nq, nkv, d, page=16):
    """Queries, a cache of 4 bits and a step's context on the host, as the attention's launches are made from them."""
    from qwen3_runtime_amd.parts.base import CacheView, GroupView, StepContext
    from qwen3_runtime_amd.parts.plan import CacheSpec

    i32 = lambda x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    pages = sum(-(-n // page) for n in kv_lens)
    width = max(-(-n // page) for n in kv_lens)
    group = GroupView(page, None, torch.zeros(len(kv_lens), width, dtype=torch.int32), i32([0] * sum(q_lens)))
    t = {"k": torch.zeros(pages, nkv, page, d // 2, dtype=torch.uint8), "v": torch.zeros(pages, nkv, page, d // 2, dtype=torch.uint8),
         "steps": torch.zeros(pages, nkv, page, 4, dtype=torch.bfloat16)}
    cache = CacheView(CacheSpec("paged_kv", heads=nkv, head_dim=d, bits=4), group=group, k=t["k"], v=t["v"], pages=t)
    cu = [0]
    for n in q_lens:
        cu.append(cu[-1] + n)
    ctx = StepContext(ops=None, dtype=torch.bfloat16, device=torch.device("cpu"), num_tokens=cu[-1], num_seqs=len(q_lens),
                      positions=i32([n - q + i for q, n in zip(q_lens, kv_lens) for i in range(q)]), cu_q=i32(cu), kv_lens=i32(kv_lens),
                      seq_of_token=i32([s for s, q in enumerate(q_lens) for _ in range(q)]), state_slots=i32([0] * len(q_lens)),
                      first_span=i32([0] * len(q_lens)), q_lens_host=list(q_lens), kv_lens_host=list(kv_lens), max_q_len=max(q_lens),
                      max_kv_len=max(kv_lens), groups=[group])
    return torch.zeros(cu[-1], nq * d, dtype=torch.bfloat16), cache, ctx


class StubLibrary:
    """An attention library that notes what it is called with, and whether the tensor behind the parts' room is there."""

    def __init__(self, made):
        self.made, self.calls = made, []

    def qrt_attention4(self, *args):
        parts = args[9]
        held = [ref() for ref in self.made]
        self.calls.append((args, not parts or any(t is not None and t.data_ptr() == parts for t in held)))
        return 0


@pytest.fixture
def stub(monkeypatch):
    from qwen3_runtime_amd.ops import hip

    made = []
    new_empty = torch.Tensor.new_empty

    def noted(self, *args, **kwargs):
        t = new_empty(self, *args, **kwargs)
        made.append(weakref.ref(t))
        return t

    lib = StubLibrary(made)
    monkeypatch.setattr(torch.Tensor, "new_empty", noted)
    monkeypatch.setattr(hip, "attention4_library", lambda d: lib)
    monkeypatch.setattr(hip, "_stream", lambda: 0)
    monkeypatch.setattr(hip, "_need", lambda t, *a, **k: t)
    monkeypatch.setattr(hip.HipOps, "_check_cache4", staticmethod(lambda cache, nkv, d: cache.k.shape[0]))
    return lib


@pytest.mark.parametrize("q_lens,kv_lens", [([1], [4000]), ([40, 1], [60, 4000]), ([24], [9000])])
def test_the_room_for_parts_lives_until_the_launches_are_made(stub, q_lens, kv_lens):
    """Freed before, it could be another thread's on the same stream, or gone, when the kernels write it."""
    from qwen3_runtime_amd.ops.hip import HipOps

    q, cache, ctx = host_step(q_lens, kv_lens, 8, 2, 64)
    HipOps()._attention4(q, cache, ctx, 8, 2, 64, 0.125, 0, 0, 0.0, 0, False)
    assert any(args[9] for args, _ in stub.calls)  # some launch of each of these steps takes its keys in pieces
    assert all(held for _, held in stub.calls)


def test_a_step_whose_lengths_have_grown_is_planned_again(stub):
    """The same context with longer contexts in it: as many keys as there are now, and a block table that has room for them."""
    from ctypes import sizeof

    from qwen3_runtime_amd.ops.hip import HipOps, OpsError, _Attn4Plan

    o = HipOps()
    q, cache, ctx = host_step([1, 1], [1500, 100], 8, 2, 64)
    attend = lambda: o._attention4(q, cache, ctx, 8, 2, 64, 0.125, 0, 0, 0.0, 0, False)  # noqa: E731

    def reach():
        plan = _Attn4Plan.from_buffer_copy(stub.calls[-1][0][0][:sizeof(_Attn4Plan)])
        return 32 * plan.piece * plan.pieces

    ctx.kv_lens_host, ctx.max_kv_len = [90, 100], 100
    attend()
    first = reach()
    ctx.kv_lens_host, ctx.max_kv_len = [1500, 100], 1500
    attend()
    assert 100 <= first < 1500 <= reach()
    ctx.kv_lens_host, ctx.max_kv_len = [1500, 100], 1505  # the longest that is said to come counts
    with pytest.raises(OpsError, match="pages wide"):
        attend()


@pytest.mark.parametrize("scale,softcap", [(float("nan"), 0.0), (float("inf"), 0.0), (0.1, float("inf")), (0.1, float("nan")), (0.1, -1.0)])
def test_scales_and_caps_that_make_no_numbers_are_refused(stub, scale, softcap):
    """Scores over an infinite cap are 0, and it times their tangent NaN."""
    from qwen3_runtime_amd.ops.hip import HipOps, OpsError

    q, cache, ctx = host_step([1], [50], 4, 2, 64)
    with pytest.raises(OpsError):
        HipOps()._attention4(q, cache, ctx, 4, 2, 64, scale, 0, 0, softcap, 0, False)
    assert not stub.calls


# ---- what a loader holds


class Table:
    """A source of random tensors for a model's declarations."""

    def __init__(self, model, seed=0):
        self.t = {}
        for i, d in enumerate(model.tensor_decls()):
            g = torch.Generator().manual_seed(seed + i)
            self.t[d.file_name] = (torch.randint(0, 4, d.shape, generator=g, dtype=torch.int32) if d.storage == "int" else
                                   torch.randn(d.shape, generator=g).to(torch.bfloat16))

    def names(self):
        return list(self.t)

    def has(self, name):
        return name in self.t

    def shape(self, name):
        return tuple(self.t[name].shape)

    def dtype(self, name):
        return self.t[name].dtype

    def get(self, name, device):
        return self.t[name].to(device)


@pytest.mark.parametrize("name", ["dekinex_tiny_a", "dekinex_tiny_b", "tiny_b", "deginex_tiny_a", "sarudra_tiny_b"])
def test_no_floats_stay_beside_their_8_bits(name):
    """Also where a part makes its matrix of what it loads: queries and keys that turn in pairs of neighbours have their rows in another order."""
    from qwen3_runtime_amd.engine.factory import build_model
    from qwen3_runtime_amd.registry import preset_config
    from qwen3_runtime_amd.weights import load_model

    whole, model = build_model(preset_config(name))[1], build_model(preset_config(name))[1]
    source = Table(whole)
    floats = load_model(whole, source, "cpu", torch.bfloat16)
    loader = load_model(model, source, "cpu", torch.bfloat16, weights="int8")
    # what the parts with matrices in 8 bits ask for in floats is not held, and what they hold is counted in its place
    parts = [p for p in model.parts() if p.int8_products]
    matrices = {d.file_name: 2 * d.shape[0] * d.shape[1] for p in parts for d in p.tensor_decls() if d.init == "matrix" and len(d.shape) == 2}
    left = [key for key in loader._cache if key[0] in ("matrix", "fused") and matrices.keys() & {key[1]} | matrices.keys() & set(key[1])]
    assert parts and not left
    coded = sum(getattr(p, n).num_bytes for p in parts for n in p.int8_products)
    assert loader.num_bytes == floats.num_bytes - sum(matrices.values()) + coded


def test_a_model_without_a_part_that_has_8_bits_is_refused():
    """Layers of memory and experts alone, one of them shared."""
    import copy

    from qwen3_runtime_amd.engine.factory import build_model
    from qwen3_runtime_amd.registry import preset_config
    from qwen3_runtime_amd.weights import load_model

    raw = copy.deepcopy(preset_config("dekinex_tiny_a"))
    memory, attention = raw["layers"][0], raw["layers"][1]
    raw["layers"] = [{**memory, "mlp": attention["mlp"]}]
    del raw["loop"]
    load_model(model := build_model(raw)[1], Table(model), "cpu", torch.bfloat16)
    with pytest.raises(ValueError, match="no attention over keys and values and no dense feed-forward"):
        load_model(model := build_model(raw)[1], Table(model), "cpu", torch.bfloat16, weights="int8")


def test_a_matrix_that_another_part_holds_as_floats_stays():
    from qwen3_runtime_amd.ops import Int8Weight
    from qwen3_runtime_amd.weights.loader import WeightLoader

    class Holder:
        def __init__(self, *names):
            self.int8_products, self.tensor_names = names, {"w": "w"}

        def load(self, fetch):
            self.w = fetch.matrix("w")

    class Source:
        def get(self, name, device):
            return torch.ones(4, 128, dtype=torch.bfloat16)

    for order in ((Holder(), Holder("w"), Holder("w")), (Holder("w"), Holder("w"), Holder())):
        loader = WeightLoader(Source(), "cpu", torch.bfloat16)
        for part in order:
            part.load(loader)
            loader.quantize(part)
        coded = [p.w for p in order if p.int8_products]
        assert all(isinstance(w, Int8Weight) for w in coded) and coded[0] is coded[1]
        assert loader.num_bytes == 4 * 128 * 2 + coded[0].num_bytes


# ---- launches of captured steps


def test_a_graphs_pieces_follow_from_its_key():
    """Whatever lengths a graph has met first: the key is all that its launches are shaped by, and lengths of one key are no more than 1.5 apart."""
    from qwen3_runtime_amd.engine.graph import DecodeGraph
    from qwen3_runtime_amd.ops.hip import HipOps

    for batch in (1, 2, 8, 64):
        for unequal in (False, True):
            for max_kv in (1, 400, 512, 513, 768, 769, 1024, 1536, 1537, 2049, 4096, 30000):
                key = DecodeGraph.key_for(batch, max_kv, True, unequal, True)
                typical = DecodeGraph.typical_lens(key)
                assert len(typical) == batch and key[1] >= max_kv and max(typical) <= key[1]
                if key[1] > 512:
                    assert DecodeGraph.key_for(batch, max(typical), True, unequal, True) == key
                    assert 0.75 <= max(typical) / max_kv <= 1.25
                # as many pieces as the same lengths get uncaptured, in a launch that has room for the bucket's
                bucket, blocks = key[1] // 32, [-(-n // 32) for n in typical]
                piece = HipOps.choose_attention4_piece(bucket, blocks, batch, 8, True)
                assert 1 <= piece <= bucket and -(-bucket // piece) <= 1024
    # without a cache of 4 bits, and up to 512 keys, there is one key a bucket
    assert DecodeGraph.key_for(4, 1000, True) == DecodeGraph.key_for(4, 600, True)
    assert DecodeGraph.key_for(4, 512, True, by_quarter=True) == DecodeGraph.key_for(4, 1, True, by_quarter=True)
    assert DecodeGraph.key_for(4, 800, False) is None


@GPU
@pytest.mark.parametrize("before,length", [(520, 900), (900, 520), (530, 740)])
def test_a_step_is_the_same_whatever_its_engine_has_served(model_folders, before, length):
    """Requests of other lengths of the same bucket come first, in one engine and not in the other: the same bits."""
    import traces
    from test_few_bits_engine import loaded

    def tail(rid, n, seed):
        toks = traces.make_requests(384, [n], seed=seed)
        return traces.tail_one_by_one({rid: next(iter(toks.values()))}, tail=4)

    def run(*steps):
        return traces.replay(loaded(model_folders["tiny_b"], 8, 256, "bfloat16", "cuda:0", cache_bits=4, hip_graph=True), traces._number([s for x in steps for s in x]))

    alone, after = run(tail("b", length, 2)), run(tail("a", before, 1), tail("b", length, 2))
    for key, want in alone.items():
        assert (want == after[key]).all(), key


@GPU
def test_decoding_across_the_quarters_of_a_bucket(model_folders):
    """Steps that leave a graph's quarter, prepared and launched ahead of their ids: the tokens of an engine without graphs."""
    from qwen3_runtime_amd import LLM, SamplingParams

    prompts = [torch.randint(0, 384, (n,), generator=torch.Generator().manual_seed(n)).tolist() for n in (757, 500)]
    made = [LLM(str(model_folders["tiny_b"]), dtype="float32", block_size=8, cache_bits=4, max_num_seqs=4, cuda_graph=graph).generate(
        prompts, SamplingParams(temperature=0.0), max_tokens=30) for graph in (True, False)]
    assert made[0] == made[1] and [len(x) for x in made[0]] == [30, 30]


# ---- rows longer than a block's registers


@GPU
@pytest.mark.parametrize("m,k", [(9, 16384), (9, 25600), (300, 12288), (300, 25600), (3, 8193), (300, 9001), (2, 1 << 17)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_codes_of_rows_that_are_read_twice(m, k, dtype):
    from test_int8_gpu import codes_of, ops, rnd

    x = rnd(m, k, seed=k, dtype=dtype)
    x[1, -1] = -1000
    got, scale = ops().quantize_rows(x)
    q, s = codes_of(x)
    assert torch.equal(got[:, :k].float(), q) and not got[:, k:].any() and torch.equal(scale, s)


@GPU
@pytest.mark.parametrize("m", [1, 4, 17, 70])
@pytest.mark.parametrize("n,k", [(5120, 25600), (40, 1 << 17)])
def test_products_of_long_rows(m, n, k):
    from test_int8_gpu import near, ops, product, rnd
    from qwen3_runtime_amd.ops import Int8Weight

    x, w = rnd(m, k, seed=m, dtype=torch.bfloat16), Int8Weight.quantize(rnd(n, k, seed=n))
    near(ops().linear(x, w), product(x, w), torch.bfloat16)
    near(ops().linear_for_residual(x, w), product(x, w), torch.float32)
