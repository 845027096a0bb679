"""What the engine's steps over the 4-bit K/V pool keep and share, on the CPU."""
import torch


def test_slots_of_a_step_stay_where_a_captured_graph_has_them(monkeypatch):
    """A longer step neither moves nor frees what shorter ones were given."""
    from minisglang_rdna4_b200.layers import attention

    monkeypatch.setattr(attention, "_COUNTING", {})
    device = torch.device("cpu")
    first = attention._counting(8, device).data_ptr()
    for n in (16384, 16385, 40000, 10, 200000):
        assert torch.equal(attention._counting(n, device), torch.arange(n, dtype=torch.int32))
        assert attention._counting(8, device).data_ptr() == first
    middle = attention._counting(17000, device).data_ptr()
    attention._counting(300000, device)
    assert attention._counting(17000, device).data_ptr() == middle != first
