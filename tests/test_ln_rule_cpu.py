"""How many partial rows the layer norm's backward writes (no GPU): its workspace is two fp32 rows for each."""
import pytest

from tossctr import _lib


@pytest.mark.parametrize("m,n,parts", [
    (512, 32, 1), (513, 32, 9), (64, 256, 1), (65, 256, 9), (32, 512, 1), (33, 512, 9),       # up to eight rows in turn
    (16, 513, 1), (16, 1024, 1), (17, 1024, 5), (32, 1024, 8), (32, 700, 8),                  # above 512 columns: four
    (1, 2048, 1), (8, 2048, 8), (4096, 2048, 1024)])
def test_partial_rows(m, n, parts):
    assert _lib.query("ctr_ln_bwd_ws_size", m, n) == 2 * parts * n * 4
