"""What the sources that reach the GPU may not hold, read as text (no GPU)."""
import glob
import os

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(REPO, "i-admm-lstm_amd")


def hip_sources():
    """The library's sources and the tools' variants of them."""
    found = [f for d in (os.path.join(PKG, "csrc"), os.path.join(REPO, "tools"))
             for e in ("*.hip", "*.h", "*.cpp") for f in glob.glob(os.path.join(d, e))]
    assert len(found) > 15
    return found


def test_every_stream_has_the_default_priority():
    """Work on streams of different priorities has hung on this hardware's runtime."""
    for path in hip_sources():
        with open(path) as f:
            text = f.read()
        assert "hipStreamCreateWithPriority" not in text, path
