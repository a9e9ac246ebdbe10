"""Lists that are shorter than the count beside them are refused before the C side reads behind them, and lists that have a
tensor twice where it would be written twice."""
import pytest
import torch

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


def clip(lengths, src, dst):
    n = len(lengths)
    D.gradClip([0], 1, n, [D.F32] * n, lengths, src, dst, 1.0, 1e-6, 3 * P, 7 * P, 1 << 40)


@pytest.mark.parametrize("lengths,src,dst,message", [
    ([4, 5, 6], [P, 2 * P, P], [P, 2 * P, P], r"dst\[0\] and dst\[2\]"),                    # in place, one gradient twice
    ([4, 5], [P, 2 * P], [4 * P, 4 * P], r"dst\[0\] and dst\[1\]"),
    ([4, 0, 5], [P, 2 * P, 3 * P], [2 * P, 2 * P, P], r"dst\[2\] shares its address with src\[0\]"),
    ([4] * 3000, [P + 64 * i for i in range(3000)], [P + 64 * i for i in range(2999)] + [P + 64 * 7], r"dst\[7\] and dst\[2999\]"),
])
def test_gradClip_refuses_a_tensor_that_would_be_written_twice(lengths, src, dst, message):
    with pytest.raises(pkg.AlphaConvError, match=message):
        clip(lengths, src, dst)


@pytest.mark.parametrize("lengths,src,dst", [
    ([4, 0, 5], [P, P, 2 * P], [P, P, 2 * P]),                                  # what is empty is not written
    ([4] * 3000, [P + 64 * i for i in range(3000)], [P + 64 * i for i in range(3000)]),
    ([4, 5], [P, P], None),                                                     # the norm alone may count a tensor twice
])
def test_gradClip_takes_other_lists(lengths, src, dst):
    """(Without a device the call ends at its first launch.)"""
    if torch.cuda.is_available():
        pytest.skip("would enqueue")
    try:
        D.gradClip([0], 1, len(lengths), [D.F32] * len(lengths), lengths, src, dst, 1.0, 1e-6, 3 * P, 7 * P, 1 << 40)
    except pkg.AlphaConvError as e:
        assert "address" not in str(e)
