"""examples/paged_decode.py at the ends of its ranges: prompts longer than one call takes.

The tokens' tolerance is that of test_paged_decode_gpu.py."""
import pytest

torch = pytest.importorskip("torch")
from test_paged_decode_gpu import E, dev, network_64  # noqa: E402, F401  (fixtures)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,max_tokens", [(700, None), (130, 64), (128, 64), (65, 64), (64, 64)])
def test_prompts_longer_than_a_call(E, dev, n, max_tokens):  # noqa: F811
    """A prompt of any length within the positions is admitted, in pieces of what a call takes."""
    cfg = E.Config(n_layers=2)
    w = E.make_weights(cfg, seed=n)
    model = E.PagedDecoder(dev, cfg, w, 64, kv="bf16", **({} if max_tokens is None else dict(max_tokens=max_tokens)))
    server = E.Server(model, 64)
    prompt = torch.randint(0, cfg.vocab, (n,), generator=torch.Generator().manual_seed(n)).tolist()
    server.admit("a", prompt)
    server.step()
    model.check()
    new = server.release("a")
    assert len(new) == 2 and sorted(server.free) == list(range(64))
    want = network_64(cfg, w, prompt + new[:1], "bf16")
    for k, t in enumerate(new):
        x = want[n - 1 + k].clone()
        seen = torch.tensor(sorted(set(prompt + new[:k])), device="cuda")
        x[seen] = torch.where(x[seen] > 0, x[seen] / 1.1, x[seen] * 1.1)
        assert float(x.max() - x[t]) <= 0.03 * 6 * float(x.std()), k


def test_a_refused_prompt_leaves_the_server_as_it_was(E, dev):  # noqa: F811
    """A prompt that the free pages or a table's width do not hold, and an empty one: no stream and no page is kept."""
    cfg = E.Config(n_layers=1)
    model = E.PagedDecoder(dev, cfg, E.make_weights(cfg, seed=1), 10)
    server = E.Server(model, 10, width=8)
    server.step()                                         # no streams yet: nothing to do
    server.admit("a", [1, 2, 3])
    for prompt in (list(range(300)), list(range(8 * 16 + 1)), []):
        with pytest.raises(ValueError):
            server.admit("b", prompt)
        assert list(server.streams) == ["a"] and len(server.free) == 9
    with pytest.raises(ValueError):
        server.admit("a", [4])
    server.admit("b", list(range(100)))
    server.step()
    model.check()
    assert len(server.release("a")) == 2 and len(server.release("b")) == 2 and sorted(server.free) == list(range(10))
