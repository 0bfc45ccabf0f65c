"""What the ranks of the synthetic training example print to one stream."""
import os
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "examples"))


def test_a_line_is_one_write(monkeypatch):
    """Unbuffered, as launchers start ranks, every write goes out by itself: a line end written apart from its line comes
    behind another rank's line."""
    import cmr_synthetic

    class Stream:
        writes = []

        def write(self, s):
            self.writes.append(s)

        def flush(self):
            pass

    monkeypatch.setattr(sys, "stdout", Stream())
    cmr_synthetic.say("rank 0 weight checksum 1.0")
    monkeypatch.undo()
    assert Stream.writes == ["rank 0 weight checksum 1.0\n"]
