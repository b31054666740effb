"""GPU tests of the 8-bit cache at the borders of its kernels' ranges: rows of several blocks
of query columns, and the calls that follow on the same handle."""
import numpy as np
import pytest

from test_gpu_cache import Rig

pytestmark = pytest.mark.gpu


def single_tokens(rig):
    """The rig's rows with one query each from here on, by the same handle."""
    rig.news = rig.starts = rig.d_starts = None
    rig.tokens = rig.rows


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("d", [192, 256, 512])
@pytest.mark.parametrize("group, new", [(1, 17), (4, 6), (8, 4), (3, 11), (1, 48), (8, 6), (7, 7)])
def test_rows_of_several_blocks_of_columns(group, new, d, dtype):
    """17 to 49 columns a row in tables that the rows fill, and single tokens behind them."""
    for lengths, news in (([64], [new]), ([992, 500, 64], [new, 1, new]), ([300] * 5, [new] * 5)):
        rig = Rig(lengths, news=news, kv=1, group=group, d=d, dtype=dtype, slots=-(-max(lengths) // 16))
        rig.attend()
        rig.attend(window=40)
        single_tokens(rig)
        rig.attend()
        rig.attend(window=40)


@pytest.mark.parametrize("kv, group, new, length, d, dtype", [
    (2, 4, 6, 8100, 256, "bf16"), (2, 4, 10, 3000, 256, "f32"), (1, 8, 3, 8100, 256, "f32"),
    (1, 8, 4, 8100, 512, "bf16"), (2, 4, 8, 500, 512, "f32")])
def test_few_new_tokens_behind_long_contexts(kv, group, new, length, d, dtype):
    rig = Rig([length], news=[new], P=64, B=32, kv=kv, group=group, d=d, dtype=dtype,
              slots=8192 // 64 if length > 2000 else 9)
    for _ in range(2):
        rig.attend()
    single_tokens(rig)
    for _ in range(2):
        rig.attend()
