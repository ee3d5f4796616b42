"""Attention of hundreds of short sequences whose rows are dealt out to waves: more places of the line than a workgroup has threads, so that the line is
searched again for every item."""
import numpy as np
import pytest

from test_attention_forms_gpu import check_biased, check_cross, ctx, make_bias  # noqa: F401  (ctx: the fixture)
from test_attention_gpu import make_cache, tell

pytestmark = pytest.mark.gpu

TEXTS = [(64 + 7 * i % 65, 64 + 7 * i % 65) for i in range(400)]                     # every row of texts of 64 to 128 tokens
CHUNKS = [(i * 37 % 129, 1 + i * 53 % 100 if i % 9 else 0) for i in range(399)] + [(128, 700)]      # rows of any number, also more than tokens; a long one


@pytest.mark.parametrize("form,dim", [(form, dim) for form in ("cross", "causal", "both") for dim in (64, 96)] + [("cross", 128)])
@pytest.mark.parametrize("seqs", [TEXTS, CHUNKS], ids=["texts", "chunks"])
def test_hundreds_of_short_texts(ctx, form, seqs, dim):
    tell("apart", form, dim)
    rng = np.random.default_rng(dim)
    lens = [n for n, _ in seqs]
    kv, pages = make_cache(rng, lens, 64, 4, dim)
    q_start = np.cumsum([0] + [m for _, m in seqs])
    q = rng.standard_normal((q_start[-1], 4, dim)).astype(np.float32)
    args = ctx, kv, pages, q, q_start, lens
    most = max(m for _, m in seqs)
    if form == "cross":
        check_cross(*args, max_q=most)
    else:
        check_biased(*args, make_bias(rng, 4, 40)[0], form == "causal", max_q=most)
