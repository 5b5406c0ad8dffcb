"""The largest caches that attention over a paged cache takes: its tiles are counted in 32 bits.  No GPU: arguments are looked at before anything else."""
import ctypes as C

import pytest

import ane_amd.bridge as br
from test_paged_places import P, cache, refused

# heads, pages of 16 whose tiles (16 positions; bfloat16: 32), and 8 for each head's beginning, are at most 2^31 - 256 in all
MOST = {"": [(32, 67108848), (63, (2 ** 31 - 256) // 63 - 8), (4096, (2 ** 31 - 256) // 4096 - 8)],
        "_bf16": [(64, 67108840), (127, 2 * ((2 ** 31 - 256) // 127 - 8)), (4096, 2 * ((2 ** 31 - 256) // 4096 - 8))]}


@pytest.mark.parametrize("end", MOST)
def test_more_tiles_than_are_counted(end):
    fn = getattr(br.lib, "mi355_attn_paged%s_dev" % end)
    for kv, most in MOST[end]:
        tiles = -(-most // 2) if end else most
        assert (tiles + 8) * kv <= 2 ** 31 - 256 < (tiles + 9) * kv
        refused(fn, C.byref(cache(kv_heads=kv, max_pages=most + 1)), P, P, P, P, P, kv, 1, 1, 0.125)
        assert "tiles" in br.last_error()
