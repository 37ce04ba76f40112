"""The workspace of the layer norm's gradients: a part for every block that makes one."""

from yabt_amd import _lib


def test_workspace_of_long_rows():
    """Rows past the registers are summed by at most 768 blocks in all, each with
    some of the columns, so that the parts take 768 blocks' columns twice (1024
    columns of fp32 or 2048 of 16 bits a block) and one more row of them."""
    size = _lib.load().yabt_layer_norm_grad_workspace_bytes
    for n, D in ((3000, 1_000_000), (100_000, 40_000), (5, 3_000_000), (1_000_000, 17_000)):
        assert 8 * D <= size(n, D) <= 8 * (768 * 2048 + D), (n, D, size(n, D))


def test_workspace_grows_with_the_rows():
    size = _lib.load().yabt_layer_norm_grad_workspace_bytes
    for D in (1, 7, 100, 513, 4096, 16_384, 16_385, 20_000, 1_000_000):
        sizes = [size(n, D) for n in (0, 1, 5, 33, 100, 1000, 4000, 100_000, 10_000_000)]
        assert sizes == sorted(sizes) and sizes[0] >= 8 * D and sizes[-1] <= 768 * 8 * D
