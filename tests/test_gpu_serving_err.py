"""The error words of the serving operators: which tensors are taken for one, and what reads them."""
import pytest

torch = pytest.importorskip("torch")

from rustane_b200 import RustaneError, ops  # noqa: E402
from test_gpu_serving import rope_case  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("err", [lambda: torch.zeros(1, dtype=torch.int32), lambda: torch.zeros(1, dtype=torch.int64, device="cuda"),
                                 lambda: torch.zeros(0, dtype=torch.int32, device="cuda"), lambda: torch.zeros(1, device="cuda")])
def test_err_has_to_be_a_word_on_the_device(err):
    _, qkv, pos, rope, _, _ = rope_case(4, 2, 2, 64, 64, "half", False, seed=0)
    for call in (lambda: ops.qk_norm_rope(qkv, pos, rope, 2, 2, err=err()),
                 lambda: ops.qk_norm_rope_backward(qkv, None, pos, rope, 2, 2, err=err()),
                 lambda: ops.logits_adjust(qkv.float(), err=err())):
        with pytest.raises(ValueError, match="err"):
            call()


def test_check_waits_for_calls_of_other_streams():
    """A call on another stream, still to come when check() is called, is one of the calls so far."""
    _, qkv, pos, rope, _, _ = rope_case(4, 2, 2, 64, 64, "half", False, seed=0)
    cache = ops.KvCache.empty(2, 16, 2, 64, torch.bfloat16, "cuda")
    slots = torch.tensor([0, 1, 32, 2], dtype=torch.int32, device="cuda")
    good = torch.arange(4, dtype=torch.int32, device="cuda")
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        ops.kv_append(qkv, pos, good, rope, cache, 2)  # the stream's first call loads and allocates, which waits
        side.synchronize()
        torch.cuda._sleep(100_000_000)  # some 50 ms
        ops.kv_append(qkv, pos, slots, rope, cache, 2)
    with pytest.raises(RustaneError):
        cache.check()
    cache.check()
