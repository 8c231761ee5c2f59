"""attention_fwd refuses what its kernel would read past: other shapes, types or devices than those it names."""
import pytest
import torch


def test_forward_refusals(native_lib):
    from pipelink_b200 import attention
    z = lambda *s, dtype=torch.bfloat16: torch.zeros(*s, dtype=dtype)
    q, k = z(1, 128, 4, 128), z(1, 128, 2, 128)
    for a in ((q, k, k), (q[0], k, k), (q[..., :64], k, k), (q[:, :0], k[:, :0], k[:, :0]), (q, k[:, :64], k[:, :64]),
              (q, k, k[:, :, :1]), (q, k.float(), k), (q.float(), k, k), (q, k[..., :64], k[..., :64]), (q, z(1, 128, 3, 128), z(1, 128, 3, 128))):
        with pytest.raises(ValueError):
            attention.attention_fwd(*a)


def test_work_lists_stay_with_the_graphs_that_read_them():
    """A list that later shapes pushed out of the cache would be freed memory to a graph captured with it."""
    from pipelink_b200 import attention
    first = attention._device_work(1, 128, 2, 2, 0, "cpu")
    for n in range(2, 300):
        attention._device_work(1, 128, 2 * n, 2, 0, "cpu")
    assert attention._device_work(1, 128, 2, 2, 0, "cpu") is first
