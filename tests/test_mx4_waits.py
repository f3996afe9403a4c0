"""The bounded waits of the MXFP4 product: what an expired one leaves behind. No GPU fault, trap or hang is involved."""
import pytest
import torch

from test_mx4 import close, linear_ref, op64, rnd, weight

pytestmark = pytest.mark.gpu

# every form of the product: fused (plain x, few tiles), 64-wide, 128-wide, CTA pairs; and one tile of very long rows, whose
# waits last a millisecond
FORMS = {"fused": (300, 128, 320), "narrow": (1000, 192, 640), "wide": (20001, 160, 320), "pair": (20001, 200, 1800),
         "long rows": (16, 8, 1 << 20)}


@pytest.mark.parametrize("form", list(FORMS))
def test_earlier_code_in_the_error_word_does_not_end_a_product(sdg, cuda, form):
    M, N, K = FORMS[form]
    wc, ws = weight(sdg, N, K, 1)
    x, res = rnd(M, K, seed=2, dtype=torch.float16), rnd(M, N, seed=3, dtype=torch.float16)
    xq = sdg.quantize_mx4(x)
    word = torch.full((1,), 0x101, dtype=torch.int32, device=cuda)
    clean = torch.zeros(1, dtype=torch.int32, device=cuda)
    ref, d = linear_ref(op64(*xq, K), op64(wc, ws, K), None, res, 0)
    for err in (word, clean):
        for y in (sdg.linear_mx4(x, wc, ws, residual=res, err_word=err),
                  sdg.linear_mx4(xq[0], wc, ws, residual=res, xscale=xq[1], err_word=err)):
            close(y, ref, d)
    assert int(word) == 0x101 and int(clean) == 0
