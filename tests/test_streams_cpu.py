"""CPU: the library's own streams."""
import os
import re

from pdae_amd import build as B


def test_no_stream_has_a_priority_of_its_own():
    """Work on streams of different priorities can stop for good on this hardware: every stream is made with the default one, in the sources and in Python."""
    root = os.path.dirname(B.HERE)
    paths = [os.path.join(B.CSRC, f) for f in os.listdir(B.CSRC)] + [os.path.join(d, f) for d, _, fs in os.walk(B.HERE) for f in fs if f.endswith(".py")] + [os.path.join(root, "bench.py")]
    for p in paths:
        with open(p, errors="replace") as f:
            text = f.read()
        assert not re.search(r"StreamCreateWithPriority|Stream\([^)]*priority\s*=|is_high_priority_stream\s*=\s*True", text), p
