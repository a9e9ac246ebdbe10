"""Lists that are shorter than the count beside them are refused before the C side reads behind them."""
import pytest

from util import load_package

pkg = load_package()
D = pkg.Cuda_dense
P = 1 << 20          # never dereferenced


@pytest.mark.parametrize("name", ["types", "lengths", "src", "dst"])
def test_gradClip_lists_shorter_than_the_count(name):
    a = dict(types=[D.F32, D.F32], lengths=[4, 5], src=[P, 2 * P], dst=[P, 2 * P])
    a[name] = a[name][:1]
    with pytest.raises(pkg.AlphaConvError, match="shorter than the count 2"):
        D.gradClip([0], 1, 2, a["types"], a["lengths"], a["src"], a["dst"], 1.0, 1e-6, 3 * P, 7 * P, 1 << 40)


def test_gradClip_workspace_of_a_short_list():
    with pytest.raises(pkg.AlphaConvError, match="shorter than the count 3"):
        D.gradClip_workspace(3, [1, 2])
    assert D.gradClip_workspace(1, [1, 2]) == D.gradClip_workspace(1, [1])


def test_streams_shorter_than_their_length():
    with pytest.raises(pkg.AlphaConvError, match="0 streams given, length 1"):
        D.matMul_fused([], 1, D.F32, P, 8, 2 * P, 8, 0, 0, 0.0, 0, 0, 0, 0, 3 * P, 8, 8, 8, 8, 0, 0)
