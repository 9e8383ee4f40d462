"""The example layer (int8 projections around rotary, cache and attention)
gives the same result token by token as in one pass, and the result that
plain 64-bit attention gives on the layer's own int8 projections."""
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "examples"))

import attention_oracle as ref  # noqa: E402


def test_example_layer_step_by_step():
    import attention_layer
    assert attention_layer.main() <= 1


def test_example_layer_against_plain_attention(ctx):
    import attention_layer
    layer = attention_layer.AttentionLayer(ctx, q_heads=6, kv_heads=3, dim=64, seed=5)
    n = 70
    layer.add_sequence(n)
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randint(-127, 128, (n, layer.width), generator=g, dtype=torch.int8, device="cuda")
    mixed, _ = layer(x, [n])
    h = layer.qkv(x, 0)
    torch.cuda.synchronize()
    h = h.view(n, 12, 64).double() * layer.scale_qkv
    bits = attention_layer.attention.rotary_frequencies(layer.rotary.desc)
    freq = torch.tensor([int(b) / 2.0 ** 64 * 2 * torch.pi for b in bits], dtype=torch.float64)
    pos = torch.arange(n, device="cuda")
    # The cache and q hold the turned heads in F16.
    q = ref.rotate(h[:, :6], pos, 64, "half", freq).half()
    k = ref.rotate(h[:, 6:9], pos, 64, "half", freq).half()
    out, _, tol, _ = ref.attend(q, k, h[:, 9:].half(), 0, True, 0, 64 ** -0.5)
    want = (out / layer.scale_attn).clamp(-128, 127)
    # A rounding of q or k to the other F16 neighbour (2^-11 of it) moves a score by at most
    # 2^-10 sum|q||k| / 8; weights move by twice that at most.
    move = 2.0 ** -9 * torch.einsum("thd,jhd->thj", q.double().abs(),
                                    k.double().abs().repeat_interleave(2, 1)).amax(2) / 8
    slack = (tol + move[..., None] * h[:, 9:].abs().max()) / layer.scale_attn + 0.5 + 1e-3
    assert ((mixed.view(n, 6, 64).double() - want).abs() <= slack).all()
