"""What a kernel's status word says when it is read."""
import pytest
import torch

from shift_b200.ops import _ext


@pytest.mark.parametrize("code,text", [(1, "wait expired"), (2, "wait expired"), (3, "offsets on the device"), (9, "unknown")])
def test_each_code_has_its_text(monkeypatch, code, text):
    word = torch.zeros(16, dtype=torch.int32)
    word[0] = code
    monkeypatch.setattr(_ext, "_status", {0: word})
    with pytest.raises(RuntimeError, match=text) as e:
        _ext.check_status(torch.device("cuda", 0))
    assert f"status {code}" in str(e.value) and ("wait" in str(e.value)) == (code in (1, 2))
    assert _ext.check_status(torch.device("cuda", 0)) == 0       # it was cleared
