"""The error words of the serving operators: which tensors are taken for one, and what reads them."""
import pytest

torch = pytest.importorskip("torch")

from rustane_b200 import ops  # noqa: E402
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
