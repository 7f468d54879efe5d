"""What the feed-forward block asks for beside its operands."""
import pytest


@pytest.mark.parametrize("kind", [0, 2, 3], ids=["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("back", [0, 1])
@pytest.mark.parametrize("c,hidden,out", [(16, 65536, 16), (65536, 65536, 65536), (65536, 16, 16), (16, 16, 65536), (512, 2048, 512), (100, 8191, 36), (33, 30000, 7)])
def test_scratch_of_the_rows_is_bounded_at_any_width(kind, back, c, hidden, out):
    """The rows' part is at most 2^30 bytes and the shares of split sums 2^27, whatever the widths and the rows."""
    from ss_conv import _ext
    planes = 3 if kind == 0 else 1
    pitch = lambda w: -(-w // 16) * 16  # noqa: E731
    weights = (2 * hidden * pitch(c) + out * pitch(hidden)) * 2 * planes + (4 * (2 * hidden * c + out * hidden) if back else 0)
    for n in (300, 4097, 2 ** 20, 2 ** 30):
        got = int(_ext.lib().ssc_gated_ff_scratch_bytes(kind, n, c, hidden, out, back))
        assert 0 < got <= 2 ** 30 + 2 ** 27 + weights, (n, got, weights)
