"""The experts' layer where torch's allocator has no room for its workspace."""
import pytest

from test_gpu_mx4_moe import D, FL, Layer, activations, gen

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def test_no_room_for_the_workspace():
    """torch's own error, which a program catches to try a smaller batch; afterwards the call works again."""
    g = gen(31)
    layer = Layer(2, 2, 64, 4096, g)
    x = activations(64, 64, FL, g)
    want = layer.check(x)[0]
    out = torch.zeros_like(x)
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    total = torch.cuda.get_device_properties(0).total_memory
    kept = []
    try:
        torch.cuda.set_per_process_memory_fraction(torch.cuda.memory_reserved() / total)
        for k in range(36, 19, -1):  # what is reserved and free, of whatever ran before
            try:
                while True:
                    kept.append(torch.empty(1 << k, dtype=torch.uint8, device=D))
            except torch.OutOfMemoryError:
                pass
        with pytest.raises(torch.OutOfMemoryError):
            layer(x, out)
    finally:
        torch.cuda.set_per_process_memory_fraction(1.0)
        del kept
    assert not out.any()
    assert torch.equal(layer(x, out)[0], want)
