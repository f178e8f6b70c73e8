"""Paged caches and rotary positions at the edges of what their calls document, without a GPU."""
import re
from pathlib import Path

CSRC = Path(__file__).resolve().parent.parent / "pallas-flexattn_b200" / "csrc"


def test_a_wait_that_gave_up_is_reported_whichever_warp_it_was():
    """No wait can be made to run out from outside, so this reads the source: the timeout is reported behind the
    barrier that all warps of a CTA reach after their last wait, and every wait's failure sets the flag."""
    src = (CSRC / "fa_paged.cu").read_text()
    kernel = src[src.index("paged_attn_kernel("):src.index("int sm_count()")]
    report = kernel.index("report_status(a.status, FA_ERR_TIMEOUT)")
    waits = [m.start() for m in re.finditer(r"\b(?:wait_for|wait_for_w|mbar_wait_w|mbar_try_wait)\(", kernel)]
    assert len(waits) > 15 and kernel.count("FA_ERR_TIMEOUT") == 1
    assert "__syncthreads();" in kernel[max(waits):report]
    for at in waits:
        start = max(kernel.rindex(c, 0, at) for c in ";{}") + 1
        used = kernel[start:at].strip()
        assert used, f"a wait whose result is dropped: {kernel[at:at + 80]}"
