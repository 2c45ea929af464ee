"""The 8-bit copies of the weights that `MoKMoE` keeps between calls, with the quantizers replaced by plain copies on the CPU and the
answer to "is this stream being captured" by a switch: a capture records work and runs none of it."""
import copy
import os

import pytest
import torch


@pytest.fixture
def layer(monkeypatch):
    """A module with what its copies were last filled with: `recorded` stands for graph memory that no replay has filled."""
    import torch.distributed as dist
    import mok
    from mok import module
    own = not dist.is_initialized()
    if own:
        dist.init_process_group("gloo", init_method=f"tcp://127.0.0.1:{29911 + os.getpid() % 80}", rank=0, world_size=1)
    state = {"capturing": False, "made": 0}

    def quantize(w, *, tile_rows):
        assert tile_rows == 128
        state["made"] += 1
        codes = torch.full_like(w, float("nan")) if state["capturing"] else w.detach().clone()
        return codes, torch.ones(w.shape[0], 1, 1)
    monkeypatch.setattr(module, "quantize_blocks", quantize)
    monkeypatch.setattr(module, "quantize_routed_weights", lambda *weights: tuple(quantize(w, tile_rows=128) for w in weights))
    monkeypatch.setattr(module, "_capturing", lambda device: state["capturing"], raising=False)
    m = mok.MoKMoE(64, 64, 2, 1)
    m.state = state
    yield m
    if own:
        dist.destroy_process_group()


def _params(m):
    return m.w_routed_gate, m.w_routed_up, m.w_routed_down


def _right(m, copies):
    return all(torch.equal(c[0], p) for c, p in zip(copies, _params(m)))


def test_copies_are_kept_until_a_weight_changes(layer):
    first = layer._block_weights()
    assert _right(layer, first) and layer._block_weights() is first and layer.state["made"] == 3
    with torch.no_grad():
        layer.w_routed_up.add_(1.0)
    assert _right(layer, layer._block_weights()) and layer.state["made"] == 6
    layer.invalidate_quantized()
    assert _right(layer, layer._block_weights()) and layer.state["made"] == 9
    layer.cache_quantized = False
    assert _right(layer, layer._block_weights()) and layer.state["made"] == 12


def test_a_capture_leaves_no_copies_behind(layer):
    layer.state["capturing"] = True
    layer._block_weights()
    layer.state["capturing"] = False
    assert _right(layer, layer._block_weights())             # eager, before any replay
    with torch.no_grad():
        layer.w_routed_down.mul_(2.0)
    layer.state["capturing"] = True
    layer._block_weights()                                   # the first call after an update is captured
    layer.state["capturing"] = False
    assert _right(layer, layer._block_weights())


def test_a_captured_decode_reads_the_present_copies(layer):
    layer._block_weights()
    layer.state["capturing"] = True
    captured = layer._block_weights()                        # valid copies: read as they are
    layer.state["capturing"] = False
    assert layer.state["made"] == 3
    places = [t.data_ptr() for c in captured for t in c]
    for change in (lambda: layer.w_routed_gate.mul_(3.0), lambda: layer.invalidate_quantized()):
        with torch.no_grad():
            change()
        now = layer._block_weights()
        assert _right(layer, now) and _right(layer, captured) and [t.data_ptr() for c in now for t in c] == places


def test_new_storage_at_the_same_address_is_noticed(layer):
    memory = torch.randn(2 * 64 * 64).to(torch.bfloat16).view(torch.int16).numpy()
    with torch.no_grad():
        layer.w_routed_gate.data = torch.from_numpy(memory).view(torch.bfloat16).view(2, 64, 64)
    assert _right(layer, layer._block_weights())
    version, address = layer.w_routed_gate._version, layer.w_routed_gate.data_ptr()
    memory += 1                                              # the allocator hands the address out again
    layer.w_routed_gate.data = torch.from_numpy(memory).view(torch.bfloat16).view(2, 64, 64)
    assert (layer.w_routed_gate._version, layer.w_routed_gate.data_ptr()) == (version, address)
    assert _right(layer, layer._block_weights())


def test_a_copied_key_matches_nothing(layer):
    layer._block_weights()
    seen = layer._quantized_blocks[0]
    assert seen.still(_params(layer)) and not copy.deepcopy(seen).still(_params(layer))


def test_mxfp8_copies_of_a_capture_are_not_kept(layer):
    layer.state["capturing"] = True
    layer._quantized_weights()
    layer.state["capturing"] = False
    kept = layer._quantized_weights()
    assert _right(layer, kept) and layer._quantized_weights() is kept
    with torch.no_grad():
        layer.w_routed_gate.mul_(2.0)
    layer.state["capturing"] = True
    layer._quantized_weights()
    layer.state["capturing"] = False
    assert _right(layer, layer._quantized_weights())


@pytest.mark.parametrize("copies", ("_block_weights", "_quantized_weights"))
def test_weights_without_version_counters(layer, copies):
    """Parameters created under inference mode: every call makes copies of what they hold then."""
    import mok
    with torch.inference_mode():
        serving = mok.MoKMoE(64, 64, 2, 1)
        for _ in range(2):
            assert _right(serving, getattr(serving, copies)())
            serving.w_routed_up.add_(1.0)
        assert _right(serving, getattr(serving, copies)())


def test_copies_are_refilled_in_every_mode(layer):
    """Made by a call under inference mode, refilled outside of it, and the other way round."""
    with torch.inference_mode():
        first = layer._block_weights()
    for mode in (False, True, False):
        with torch.no_grad():
            layer.w_routed_up.add_(1.0)
        with torch.inference_mode(mode):
            assert layer._block_weights() is first
        assert _right(layer, first)


def test_mxfp8_copies_that_a_graph_reads_stay(layer):
    """A graph captured with valid copies: their memory is not handed out again when the weights change."""
    import weakref
    layer._quantized_weights()
    layer.state["capturing"] = True
    places = [weakref.ref(c[0]) for _ in range(2) for c in layer._quantized_weights()]
    layer.state["capturing"] = False
    for change in (lambda: layer.w_routed_gate.mul_(2.0), lambda: layer.invalidate_quantized()):
        with torch.no_grad():
            change()
        assert _right(layer, layer._quantized_weights())
        assert all(p() is not None for p in places)
    assert len(layer._captured) == 1
