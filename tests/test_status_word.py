"""The device status word: where it comes from, and what a capture leaves of it."""
import pytest
import torch


def test_entry_point_refuses():
    from mok import _native as nat
    assert nat.lib().mok_status_word(None) == -1


@pytest.mark.gpu
def test_first_call_of_all_is_captured(monkeypatch):
    """The word is there before the first replay, and replays leave what others have put into it."""
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    import mok
    from mok import _native as nat
    dev = torch.device("cuda", 0)
    x = torch.randn(40, 256, device=dev).to(torch.bfloat16)
    a, b = mok.quantize_blocks(x), mok.quantize_blocks(x, tile_rows=128)
    want = mok.block_matmul(a, b)
    nat.check_status(dev)
    monkeypatch.setattr(nat, "_STATUS", {})   # as in a process that has not used it
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = mok.block_matmul(a, b)
    word = nat.status_word(dev)
    assert int(word.item()) == 0 and torch.equal(mok.block_matmul(a, b), want)
    try:
        word.fill_(4)
        g.replay()
        torch.cuda.synchronize()
        assert int(word.item()) == 4
        with pytest.raises(RuntimeError, match="pipeline"):
            nat.check_status(dev)
        assert int(word.item()) == 0
    finally:
        word.zero_()
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    nat.check_status(dev)


@pytest.mark.gpu
def test_word_of_the_library():
    """An int32 on the device, the same one in every call."""
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from mok import _native as nat
    word = nat.status_word(torch.device("cuda", 0))
    assert (word.dtype, word.shape, word.device) == (torch.int32, (1,), torch.device("cuda", 0))
    address = nat.c_void_p()
    assert nat.lib().mok_status_word(nat.ctypes.byref(address)) == 0 and address.value == word.data_ptr()
