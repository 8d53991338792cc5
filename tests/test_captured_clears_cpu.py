"""No source of the library records a memset into a caller's graph: such nodes have given wrong results on replays after the first."""
import glob
import os

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_no_memset_on_a_stream():
    files = glob.glob(os.path.join(ROOT, 'advmix_amd', 'csrc', '*.hip')) + glob.glob(os.path.join(ROOT, 'advmix_amd', 'csrc', '*.h'))
    assert len(files) > 15
    assert not [f for f in files if 'hipMemsetAsync' in open(f).read()]
