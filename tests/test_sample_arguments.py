"""What lucciola.sample refuses before it calls the library: tensors that the kernel would read as
something else (int64 as pairs of int32, fp32 logits as bf16) or past their end. No GPU needed:
the checks come first, and what they pass fails for being on the CPU."""
import pytest

import lucciola as L

torch = pytest.importorskip("torch")

NAMES = ("temperature", "top_k", "top_p", "min_p", "rand_vals", "out_idx")


def arguments(batch=4, vocab=100):
    f = torch.ones(batch)
    i = torch.ones(batch, dtype=torch.int32)
    return dict(out_idx=i.clone(), logits=torch.zeros(batch, vocab, dtype=torch.bfloat16),
                rand_vals=f * 0.5, temperature=f.clone(), top_k=i.clone(), top_p=f.clone(),
                min_p=f * 0)


def refused(name, **kw):
    with pytest.raises(L.LucciolaError, match=f"lc_sample: {name} ha") as e:
        L.sample(**dict(arguments(), **kw))
    assert e.value.status == 1
    return str(e.value)


@pytest.mark.parametrize("name", NAMES)
def test_types(name):
    good = arguments()[name]
    for dtype in (torch.int64, torch.float64, torch.float16, torch.bfloat16, torch.int16):
        refused(name, **{name: good.to(dtype)})
    refused(name, **{name: good.float() if good.dtype == torch.int32 else good.int()})


@pytest.mark.parametrize("name", NAMES)
def test_strides_and_lengths(name):
    good = arguments()[name]
    refused(name, **{name: good[:3]})
    refused(name, **{name: good[:1]})
    refused(name, **{name: good[:1].expand(4)})          # one entry for all rows
    refused(name, **{name: good.repeat(2)[::2]})
    refused(name, **{name: torch.stack([good, good], 1)[:, 0]})


def test_logits():
    refused("logits", logits=torch.zeros(4, 100))
    refused("logits", logits=torch.zeros(4, 100, dtype=torch.float16))
    refused("logits", logits=torch.zeros(100, 4, dtype=torch.bfloat16).T)
    refused("logits", logits=torch.zeros(4, 200, dtype=torch.bfloat16)[:, ::2])
    with pytest.raises(ValueError):
        L.sample(**dict(arguments(), logits=torch.zeros(100, dtype=torch.bfloat16)))


def test_host_memory_that_the_gpu_cannot_read():
    assert "on the GPU" in refused("logits")
