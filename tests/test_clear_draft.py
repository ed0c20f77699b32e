"""CPU-side checks of the drafting model's own code (clear_draft.py), over hidden rows that stand in for what its kernels give."""
import pytest

from engine_loader import load_module

torch = pytest.importorskip("torch")


def model_of(hidden):
    """a model whose run gives these hidden rows"""
    draft = load_module("clear_draft").Draft
    model = draft.__new__(draft)
    model._run = lambda tokens, lengths: hidden
    return model


HIDDEN = torch.arange(4 * 5 * 3, dtype=torch.float32).reshape(4, 5, 3)


def test_prompt_gives_the_row_of_each_lanes_last_token():
    lengths = torch.tensor([1, 5, 3, 4], dtype=torch.int32)
    got = model_of(HIDDEN).prompt(torch.zeros(4, 5, dtype=torch.int64), lengths)
    assert torch.equal(got, torch.stack([HIDDEN[b, n - 1] for b, n in enumerate(lengths.tolist())]))
    assert torch.equal(model_of(HIDDEN).prompt(torch.zeros(4, 5, dtype=torch.int64)), HIDDEN[:, -1])


def test_prompt_holds_lengths_to_the_tokens_there_are():
    """as the kernels do: past the last row lies nothing that may be read"""
    lengths = torch.tensor([6, 5, 2**31 - 1, 2], dtype=torch.int32)
    got = model_of(HIDDEN).prompt(torch.zeros(4, 5, dtype=torch.int64), lengths)
    assert torch.equal(got, torch.stack([HIDDEN[0, 4], HIDDEN[1, 4], HIDDEN[2, 4], HIDDEN[3, 1]]))


@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16])
def test_prompt_gives_zeros_where_there_is_no_last_token(kind):
    hidden = (HIDDEN + 1).to(kind)
    got = model_of(hidden).prompt(torch.zeros(4, 5, dtype=torch.int64), torch.tensor([0, 2, -3, 5], dtype=torch.int32))
    assert got.dtype == kind and torch.equal(got[[1, 3]], torch.stack([hidden[1, 1], hidden[3, 4]])) and (got[[0, 2]] == 0).all()
    for lengths in (None, torch.zeros(4, dtype=torch.int32)):
        none = model_of(hidden[:, :0]).prompt(torch.zeros(4, 0, dtype=torch.int64), lengths)
        assert none.shape == (4, 3) and none.dtype == kind and (none == 0).all()


@pytest.mark.parametrize("call", ["prompt", "step"])
def test_a_model_without_states_refuses(call):
    """before the first reset; without the check no layer would run, and the embeddings come out as hidden rows"""
    draft = load_module("clear_draft")
    model = draft.Draft.__new__(draft.Draft)
    model.w_in, model.w_out, model.states, model.dtype = [None, None], [None, None], [], torch.float32
    model.embedding = torch.ones(7, 8)
    with pytest.raises(draft.clear_ops.ClearError, match="reset"):
        getattr(model, call)(torch.zeros((2, 3) if call == "prompt" else 2, dtype=torch.int64))


def test_generate_of_no_tokens_gives_none():
    model = model_of(HIDDEN)
    model.reset = lambda lanes: None
    out = model.generate(torch.zeros(4, 5, dtype=torch.int64), 0, torch.zeros(0, 4))
    assert out.shape == (4, 0) and out.dtype == torch.int64
