"""The example that fits a query adapter: residual blocks, the loss over a corpus and the matrix steps in one training loop, whose
result is searched in a graph that was built before it."""
import os

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_adapter_brings_back_what_the_new_encoder_lost(monkeypatch):
    monkeypatch.syspath_prepend(os.path.join(ROOT, "allan-poe_amd", "examples"))
    import query_adapter
    out = query_adapter.main(["--docs", "6000", "--train", "8192", "--held-out", "256", "--steps", "80", "--batch", "257"])
    assert out["recall_at_10_old_encoder"] > 0.95                        # the graph finds what a fitting query asks for
    assert out["loss_last"] < out["loss_first"] - 1.0
    assert out["recall_at_10_after"] > out["recall_at_10_before"] + 0.1  # on queries that were held out
