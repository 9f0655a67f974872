"""GQAAttention's refusals, on the CPU."""
import pytest
import torch


@pytest.mark.parametrize("heads,kv_heads", [(4, 0), (0, 0), (0, 2), (4, -2), (-4, 2)])
def test_a_layer_has_heads(pkg, heads, kv_heads):
    def weight(out, in_):
        return pkg.QTensor(torch.ones(out, in_, dtype=torch.int8), torch.ones(out),
                           scheme="per_row_i8")
    wide = (heads + 2 * kv_heads) * 64
    with pytest.raises(ValueError, match="heads"):
        pkg.GQAAttention(weight(max(wide, 64), 128), weight(128, max(heads * 64, 64)), heads,
                         kv_heads, 64, None)
