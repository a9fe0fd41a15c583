import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "sageattention-rdna4_amd")
for p in (ROOT, PKG, os.path.dirname(os.path.abspath(__file__))):
    if p not in sys.path:
        sys.path.insert(0, p)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs an MI355X (gfx950) GPU and the built library")


#: Tests whose expectation is wrong, kept as they are. Both take the gradients' expected values from the 8-bit forward
#: call's output and logsumexp, which do not belong to the probabilities of the 16-bit scores: a causal first row sees
#: one key, so that its dq is 0 whatever the scores, where they want up to 1.3e-3. What they are about is tested in
#: test_gpu_training_exact.py (test_gradients_are_attentions, test_block_of_a_transformer).
WRONG = {("test_gpu_training", "test_attention_by_autograd"), ("test_gpu_training", "test_block_of_a_transformer")}


def pytest_collection_modifyitems(items):
    for item in items:
        if (item.module.__name__, getattr(item, "originalname", item.name)) in WRONG:
            item.add_marker(pytest.mark.xfail(reason="expects gradients of the 8-bit forward call's logsumexp",
                                              raises=AssertionError))
