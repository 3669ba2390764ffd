"""What the Python wrappers of the cache and the log probabilities look at before the C call, on tensors that only say
what they are: on the GPU, of a device and a type."""
import pytest
import torch

FLOAT, HALF, INT, CODE = torch.float32, torch.bfloat16, torch.int32, torch.uint8


class Tensor:
    is_cuda = True

    def __init__(self, dtype, device=0, values=64):
        self.dtype, self.device, self.values = dtype, device, values

    def get_device(self):
        return self.device

    def numel(self):
        return self.values

    def element_size(self):
        return self.dtype.itemsize


@pytest.fixture
def calls(monkeypatch):
    """What reached the C calls, which are not made; the current device is 0."""
    import l2c
    l2c._takes("cache_copy", "int32")  # looks up torch's types
    seen = []
    monkeypatch.setattr(l2c, "_device", lambda: 0)
    for name in ("cache_append", "cache_attention", "cache_advance", "cache_copy", "decoder_logprobs"):
        monkeypatch.setattr(l2c, "_c_" + name, lambda *args, name=name: seen.append((name, args)) or 0)
    return seen


SIZES = (8, 2, 16, 16, 4, 4, 2)
OPERATORS = {
    # wrapper, types of its tensors, what follows them, tensors by name
    "attention": ("cache_attention", (HALF, HALF, HALF, HALF, INT, INT), SIZES, dict(workspace=CODE, starts=INT)),
    "attention_e4m3": ("cache_attention", (HALF, HALF, CODE, CODE, INT, INT), SIZES,
                       dict(workspace=CODE, starts=INT, key_scales=FLOAT, value_scales=FLOAT)),
    "append": ("cache_append", (HALF, HALF, HALF, HALF, INT, INT), (2, 16, 16, 4, 4, 2), dict(starts=INT)),
    "append_e4m3": ("cache_append", (CODE, CODE, HALF, HALF, INT, INT), (2, 16, 16, 4, 4, 2),
                    dict(starts=INT, key_scales=FLOAT, value_scales=FLOAT)),
    "advance": ("cache_advance", (INT,) * 7, (2, 4, 16, 10), dict(parents=INT, starts=INT, held=INT)),
    "copy": ("cache_copy", (CODE, INT), (2, 4, 16), {}),
    "logprobs": ("decoder_logprobs", (FLOAT, FLOAT, INT, FLOAT, FLOAT, INT), (100, 2, 1), dict(workspace=CODE)),
}


def call(operator, elsewhere=None, without=()):
    """The call with one tensor, by its index or name, on device 1, or some that are None."""
    import l2c
    name, types, rest, named = OPERATORS[operator]
    make = lambda key, dtype: None if key in without else Tensor(dtype, 1 if key == elsewhere else 0)  # noqa: E731
    getattr(l2c, name)(*(make(i, t) for i, t in enumerate(types)), *rest, **{k: make(k, t) for k, t in named.items()})


@pytest.mark.parametrize("operator", OPERATORS)
def test_tensors_of_the_current_device_are_taken(calls, operator):
    call(operator)
    assert [name for name, _ in calls] == [OPERATORS[operator][0]]


@pytest.mark.parametrize("operator,which", [(o, w) for o, (_, types, _, named) in OPERATORS.items()
                                            for w in (*range(len(types)), *named)])
def test_a_tensor_of_another_device_is_refused(calls, operator, which):
    """Every one of them, the workspaces among them."""
    with pytest.raises(ValueError, match="current device"):
        call(operator, elsewhere=which)
    assert not calls


@pytest.mark.parametrize("operator,without", [
    ("logprobs", (0, 5)), ("logprobs", (1,)), ("logprobs", (2, 3)), ("logprobs", (2,)), ("logprobs", (3,)),
    ("logprobs", ("workspace",)), ("attention", ("workspace", "starts")), ("append", ("starts",)),
    ("advance", ("parents", "starts", "held")),
    ("advance", (0, 5)), ("advance", (2,)), ("advance", (0, 2, 5)),  # of no columns, of no pages
    ("copy", (0,)), ("copy", (1,)), ("copy", (0, 1)),                # of nothing
], ids=str)
def test_what_the_entry_point_may_get_as_null(calls, operator, without):
    call(operator, without=without)
    (_, args), = calls
    assert sum(a is None for a in args[:-1]) >= len(without)
