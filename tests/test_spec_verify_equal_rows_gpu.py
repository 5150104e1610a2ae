"""A refused token whose probability is 0 in the target and in an equal draft row leaves
max(p - q, 0) = 0 everywhere: the token is then drawn from p.  p - q of equal rows has to
be exactly 0 for that, whatever p is."""
import pytest
import torch

from kernels.spec_verify import speculative_verify

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("V", [1000, 1001, 20008])
@pytest.mark.parametrize("T", [1.0, 0.7])
def test_equal_rows_draw_from_the_target(dtype, V, T):
    dev = torch.device("cuda", 0)
    g = torch.Generator(device=dev).manual_seed(V)
    B = 6
    target = torch.randn(B, 2, V, device=dev, generator=g).to(dtype)
    target[:, 0, 5] = float("-inf")
    target[1, 0, 7:40] = float("nan")
    draft = target[:, :1].clone()
    noise = -torch.log1p(-torch.rand(B, V, device=dev, generator=g)) + 1e-9
    tokens, accepted, _ = speculative_verify(target, torch.full((B, 1), 5, device=dev), torch.full((B, 1), 0.5, device=dev),
                                             noise, draft, torch.full((B,), T, device=dev))
    p = (target[:, 0].double().nan_to_num(nan=float("-inf"), neginf=float("-inf")) / T).softmax(-1)
    assert accepted.tolist() == [0] * B
    assert torch.equal(tokens[:, 0], (p / noise.double()).argmax(-1))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_infinities_and_nan_of_both_rows(dtype):
    """+inf counts as the largest finite number and NaN as -inf, in the target and in the draft."""
    dev = torch.device("cuda", 0)
    g = torch.Generator(device=dev).manual_seed(3)
    B, V = 4, 2048
    target = torch.randn(B, 2, V, device=dev, generator=g).to(dtype)
    draft = torch.randn(B, 1, V, device=dev, generator=g).to(dtype)
    target[0, 0, [9, 700]] = float("inf")          # p = 1/2 at each
    draft[1, 0, ::2] = float("nan")                # q = 0 at every second token
    draft[2, 0, 11] = float("inf")                 # q = 1 at 11
    target[3, 0, 1::2] = float("nan")
    x = torch.tensor([[3], [3], [11], [3]], device=dev)
    u = torch.full((B, 1), 0.999999, device=dev)
    noise = -torch.log1p(-torch.rand(B, V, device=dev, generator=g)) + 1e-9

    def law(l):
        l = l.double().nan_to_num(nan=float("-inf"), neginf=float("-inf"), posinf=torch.finfo(torch.float32).max)
        return (l - l.max(-1, keepdim=True).values).softmax(-1)

    p, q = law(target[:, 0]), law(draft[:, 0])
    refused = u[:, 0].double() * q.gather(1, x)[:, 0] >= p.gather(1, x)[:, 0]
    tokens, accepted, _ = speculative_verify(target, x, u, noise, draft)
    assert torch.equal(accepted == 0, refused)
    want = ((p - q).clamp(min=0) / noise.double()).argmax(-1)
    assert bool(refused[0]) and bool(refused[2]) and bool(refused[3])
    assert torch.equal(tokens[:, 0][refused], want[refused])
