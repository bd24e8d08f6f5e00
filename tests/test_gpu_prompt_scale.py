"""spinn_hip_prompt_attention with the least and the largest scales over scores that show them."""
import pytest

from tests.decodeops import BF16, F32, NAMES, gen
from tests.promptops import Prompt
from tests.test_gpu_prompt import check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [F32, BF16], ids=NAMES.get)
@pytest.mark.parametrize("causal", [1, 0], ids=["causal", "full"])
@pytest.mark.parametrize("lens,kv_lens", [([40, 150], None), ([3], [5000])], ids=["whole", "split"])
def test_no_scale_over_large_scores(hip, dtype, causal, lens, kv_lens):
    """A scale of zero leaves equal weights whatever q.k is, up to 5e37 here."""
    p = Prompt(gen(1), dtype, lens, 2, 1, 64, kv_lens=kv_lens)
    p.q.mul_(1e18)
    p.k.mul_(1e18)
    check(hip, p, 0.0, causal, what="no scale")
