"""examples/train_and_search.py: the layer norm and the cross entropy train a
table of vectors, which the kNN engine then searches."""
import importlib.util
import os

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.gpu
def test_trained_table_is_searched(gpu):
    spec = importlib.util.spec_from_file_location("train_and_search", os.path.join(ROOT, "examples", "train_and_search.py"))
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    # Untrained, a query's item is among 10 of 2,000 by chance (0.5 %) and the
    # loss is about log 2,000 = 7.6; the training has to move both far.
    first, last, hit = example.main(items=2000, dim=64, batch=512, steps=150, quiet=True)
    assert first > 6.0 and last < 0.5 * first and hit > 0.5
