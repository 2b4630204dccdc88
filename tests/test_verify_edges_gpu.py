"""tree_verify on the GPU at the ends of what it takes: vocabularies past 2^20 entries, whose
chunks are longer, more sequences than workgroups are aimed at, and trees whose nodes are
all rejected."""
import pytest
import torch

from test_verify_gpu import check, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["probs", "distinct", "lookup"])
@pytest.mark.parametrize("V,dt", [(1 << 20, "f16"), ((1 << 20) + 1, "f32"), ((1 << 21) + 4097, "bf16")])
def test_large_vocabularies(dev, kind, V, dt):
    p, q, tok, u, par = make(dev, 2, 4, V, dt, 3, kind, seed=V % 1000)
    for last in (0.0, 0.37, 1 - 2.0 ** -24):
        u[:, -1] = last
        check(p, q, tok, u, par, None, kind == "distinct")


@pytest.mark.parametrize("kind", ["probs", "lookup"])
def test_more_sequences_than_workgroups(dev, kind):
    p, q, tok, u, par = make(dev, 700, 3, 1500, "f32", 2, kind, seed=7)
    check(p, q, tok, u, par)


@pytest.mark.parametrize("kind", ["probs", "distinct", "lookup"])
@pytest.mark.parametrize("T", [65, 500, 1024])
def test_every_node_is_rejected(dev, kind, T):
    """Children of the sequence that the target gives nothing, each token several times:
    what is left is the target's row."""
    V = 2100
    p = torch.zeros(2, T + 1, V, device=dev)
    p[:, :, 300:] = 1 / (V - 300)
    q = torch.zeros(2, T, V, device=dev)
    q[:, :, :300] = 1 / 300
    tok = (torch.arange(T, device=dev).int() * 7 % 300).expand(2, T).contiguous()
    u = torch.rand(2, T + 1, device=dev, generator=torch.Generator(device=dev).manual_seed(T))
    par = torch.full((2, T), -1, dtype=torch.int32, device=dev)
    _, count, nxt = check(p, None if kind == "lookup" else q, tok, u, par, None, kind == "distinct")
    assert count.tolist() == [0, 0] and (nxt >= 300).all()
