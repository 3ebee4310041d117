"""layer_run and metadata with a shared prefix: its kernels read every token by
the rows' own block tables, whose entries below the prefix need not be set, so such
calls go to the stock layer or are refused (CPU: nothing is launched)."""
from types import SimpleNamespace

import pytest
import torch

from _util import pkg


@pytest.fixture
def seam():
    lr, att = pkg("integration.layer_run"), pkg("integration.attention")
    lr.uninstall()

    def install(stock):
        layer = SimpleNamespace(name="L0", input_norm=None, kv_cache=None)
        lr.install(SimpleNamespace(layers=[layer], final_norm=None, cos_sin=None, scale=1.0,
                                   cfg=SimpleNamespace(hidden=8)), stock_layer=stock)

    def publish(rows, **kw):
        i32 = dict(dtype=torch.int32)
        lr.set_attention_metadata(att.SplitKVDecodeMetadata(
            block_tables=torch.full((rows, 4), -1, **i32), seq_lens=torch.full((rows,), 70, **i32),
            slot_mapping=torch.zeros(rows, dtype=torch.int64), num_splits=1,
            prefix_table=torch.zeros(2, **i32), prefix_len=torch.full((1,), 64, **i32), **kw))
        x = torch.zeros((rows, 8), dtype=torch.bfloat16)
        return x, x, torch.full((rows,), 69), "L0"

    yield install, publish, lr.layer_run
    lr.uninstall()


@pytest.mark.parametrize("rows", [1, 3, 16, 17])
def test_a_shared_prefix_is_refused(seam, rows):
    install, publish, layer_run = seam
    install(None)
    with pytest.raises(ValueError, match="shared prefix"):
        layer_run(*publish(rows))


@pytest.mark.parametrize("rows", [1, 3, 17])
def test_a_shared_prefix_goes_to_the_stock_layer(seam, rows):
    install, publish, layer_run = seam
    install(lambda index, x, residual, positions: ("stock", index, x.shape[0]))
    assert layer_run(*publish(rows)) == ("stock", 0, rows)


@pytest.mark.parametrize("stock", [None, lambda *a: a])
def test_packed_rows_under_a_shared_prefix_are_refused(seam, stock):
    install, publish, layer_run = seam
    install(stock)
    with pytest.raises(ValueError, match="do not go together"):
        layer_run(*publish(3, query_start_loc=torch.arange(4, dtype=torch.int32)))
