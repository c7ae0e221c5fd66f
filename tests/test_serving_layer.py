"""CronRootAttention with rotary positions, head norms and a paged cache: what the
layer checks without a GPU."""
import pytest
import torch

import cron_root_attention as cra


def test_parameters_and_state():
    plain = cra.CronRootAttention(128, 4, n_kv_heads=2)
    assert set(plain.state_dict()) == {f"{n}_proj.weight" for n in "qkvo"}
    layer = cra.CronRootAttention(128, 4, n_kv_heads=2, rotary=cra.RotaryTable(32, 64), qk_norm=True)
    assert set(layer.state_dict()) - set(plain.state_dict()) == {"q_norm", "k_norm"}
    assert layer.q_norm.shape == (32,) and layer.half().k_norm.dtype == torch.float16


def test_cache_and_batch_belong_together():
    layer = cra.CronRootAttention(64, 2)
    table, lens = torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="belong together"):
        layer(torch.zeros(1, 1, 64), batch=cra.PagedBatch(table, lens))


def test_positions_of_a_batch():
    table = torch.zeros(3, 1, dtype=torch.int32)
    lens = torch.tensor([5, 9, 3], dtype=torch.int32)
    assert cra.PagedBatch(table, lens).positions(2).tolist() == [[3, 4], [7, 8], [1, 2]]
    cu = torch.tensor([1, 3, 3, 6], dtype=torch.int32)  # one token before, two behind, an empty sequence
    pos = cra.PagedBatch(table, lens, cu).positions(8)
    assert pos.dtype == torch.int32 and pos.tolist() == [[0, 3, 4, 0, 1, 2, 0, 0]]


def test_positions_need_rotary():
    """Positions that nothing would turn by are refused, not passed over."""
    x, pos = torch.zeros(1, 4, 64), torch.arange(4)
    for qk_norm in (False, True):
        with pytest.raises(ValueError, match="rotary"):
            cra.CronRootAttention(64, 2, qk_norm=qk_norm)(x, positions=pos)
