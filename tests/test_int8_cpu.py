"""The 8-bit products and the attention over a shared prefix run on a CUDA device only: tensors elsewhere are refused, by name."""
import pytest
import torch


def test_tensors_of_the_host_are_refused():
    from flyweight_b200.kernels import KernelError, int8
    x = torch.randn(4, 64)
    for call in (lambda: int8.rows_int8(x), lambda: int8.matrix_int8(x), lambda: int8.rmsnorm_int8(x, torch.ones(64), 1e-5),
                 lambda: int8.rows_int8(x.to(torch.float16)), lambda: int8.rows_int8(x.t())):
        with pytest.raises(KernelError, match="CUDA device"):
            call()
    for call in (lambda: int8.linear_int8(x, x, torch.float32), lambda: int8.gated_int8(x, x)):
        with pytest.raises(KernelError, match="Int8Matrix"):
            call()
    with pytest.raises(KernelError, match="leaves as"):
        int8.linear_int8(x, x, torch.float16)
    with pytest.raises(KernelError, match="unknown gate"):
        int8.gated_int8(x, x, activation="softplus")


def test_the_attention_refuses_tensors_of_the_host():
    from flyweight_b200.kernels import KernelError, attention
    i32 = torch.zeros(2, dtype=torch.int32)
    pool = torch.zeros(3, 2, 64, 16)
    with pytest.raises(KernelError, match="CUDA device"):
        attention.shared_prefix_attention(torch.zeros(2, 64), pool, pool, i32, i32, i32.view(1, 2), i32, i32[:1], 4, 0.25)


def test_the_rows_say_their_layout():
    from flyweight_b200.kernels.int8 import Int8Rows
    buffer = torch.zeros(3 * 112 + 3 * 4, dtype=torch.uint8)
    buffer[:3 * 112].view(torch.int8).view(3, 112)[:, :100] = torch.arange(100, dtype=torch.int8) - 50
    buffer[3 * 112:].view(torch.float32)[:] = torch.tensor([1.0, 0.5, 2.0])
    rows = Int8Rows(buffer, 3, 100)
    assert rows.shape == (3, 100) and rows.values.shape == (3, 112) and rows.scales.tolist() == [1.0, 0.5, 2.0]
    assert torch.equal(rows.float(), (torch.arange(100.0) - 50)[None, :] * torch.tensor([[1.0], [0.5], [2.0]]))


@pytest.mark.parametrize("tokens", [1, 3, 64, 500])
@pytest.mark.parametrize("pages", [1, 8, 9, 64, 5000])
def test_the_cut_of_the_shared_pages(tokens, pages):
    from flyweight_b200.kernels.attention import shared_prefix_splits
    for wide in (False, True):
        shared, own = shared_prefix_splits(tokens, 8, 4, 64, pages, 3, wide)
        assert own in (1, 2, 4, 8) and 0 <= shared <= min(64, pages) and (shared > 0 or wide)
        # never more blocks than fill the SMs twice over, but for the one slice that there always is
        assert shared <= 1 or shared * 8 * -(-tokens * 4 // (128 if wide else 64)) <= 2 * 148
