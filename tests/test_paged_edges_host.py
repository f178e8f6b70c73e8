"""Paged caches and rotary positions at the edges of what their calls document, without a GPU."""
import re
from pathlib import Path

import pytest
import torch

from pallas_flexattn import _lib as L
from pallas_flexattn import flash_attn as F

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


def test_a_status_word_of_a_capture_is_not_the_devices(monkeypatch):
    """A word made inside a stream capture is memory of that graph: it is never cached as the device's."""
    on = {"capturing": True}
    zeros = torch.zeros
    monkeypatch.setattr(F, "_STATUS", {})
    monkeypatch.setattr(F, "_STATUS_PTR", {})
    monkeypatch.setattr(F, "_GRAPH_STATUS", {})
    monkeypatch.setattr(F, "_capturing", lambda dev: on["capturing"])
    monkeypatch.setattr(torch, "zeros", lambda *a, device=None, **kw: zeros(*a, **kw))
    monkeypatch.setattr(torch.cuda, "current_stream", lambda dev: type("S", (), {"synchronize": lambda self: None})())
    with pytest.raises(RuntimeError, match="check_device_status"):
        F.status_ptr(0)
    graph = F.device_status("cuda:0")
    on["capturing"] = False
    word = F.device_status("cuda:0")
    assert word is not graph and F.device_status("cuda:0") is word and F.status_ptr(0) == word.data_ptr()
    on["capturing"] = True
    assert F.device_status("cuda:0") is word and F.status_ptr(0) == word.data_ptr()
    for w in (word, graph):
        w.fill_(L.FA_ERR_INVALID)
        with pytest.raises(L.FlexAttnError, match="out of range"):
            F.check_device_status("cuda:0")
        assert int(w) == 0
        F.check_device_status("cuda:0")
