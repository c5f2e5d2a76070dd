"""Orderings inside the attention kernels that no run can show to be missing
reliably: read off their sources."""
import re
from pathlib import Path

CSRC = Path(__file__).resolve().parent.parent / "drama3_offloading_b200" / "csrc"


def test_rows_cleared_in_a_slot_are_fenced_before_the_slot_goes_back():
    """The row kernel's warps clear value rows behind a sequence's end with
    ordinary shared stores; the slot is then refilled by TMA, through the async
    proxy.  Every such store is followed by a proxy fence before the warp's
    next arrival."""
    src = (CSRC / "attn_rows.cuh").read_text()
    stores = [m.end() for m in re.finditer(r"st\.shared", src)]
    assert stores
    for at in stores:
        gives = re.search(r"\bgive\(\);|mbar_arrive", src[at:]).start()
        assert "fence_proxy_async_smem();" in src[at:at + gives]
