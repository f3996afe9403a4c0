"""The bounded waits of the MXFP4 product: what an expired one leaves behind. No GPU fault, trap or hang is involved."""
import pytest
import torch

from test_mx4 import close, linear_ref, op64, rnd, weight

pytestmark = pytest.mark.gpu
SDG_ERR_DEVICE = 8

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


# ------------------------------------------------------------------ loaders that stop
# (form, M, N, K, x is plain). A CTA loads ceil(K / 256) stages a tile: fused 2 stages and 3 raw tiles for up to three tiles,
# narrow 3 stages, wide 5 for two tiles and more, pairs 8 for two tiles and more
STALLED = {"fused": (1, 8192, 320, 320, True), "narrow": (2, 1000, 192, 640, False), "wide": (3, 20001, 160, 1100, False),
           "pair": (4, 20001, 200, 1800, False)}


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("form,who,stall", [("fused", 0, 0), ("fused", 0, 1), ("fused", 0, 3), ("fused", 1, 0),
                                            ("fused", 1, 2), ("fused", 1, 4), ("narrow", 0, 0), ("narrow", 0, 2),
                                            ("wide", 0, 0), ("wide", 0, 1), ("wide", 0, 7), ("pair", 0, 0), ("pair", 0, 3),
                                            ("pair", 0, 11), ("pair", 1, 0), ("pair", 1, 5), ("pair", 1, 12)])
def test_expired_wait_reports_and_leaves_the_device_usable(sdg, cuda, form, who, stall, residual):
    """A loader that stops leaves waits that nothing ends: they run out after a millisecond, the kernel waits for its copies in
    flight and returns, the call reports it, and the next product is right."""
    f, M, N, K, plain = STALLED[form]
    wc, ws = weight(sdg, N, K, 1)
    x = rnd(M, K, seed=2, dtype=torch.float16)
    res = rnd(M, N, seed=3, dtype=torch.float16) if residual else None
    xc, xs = sdg.quantize_mx4(x)
    want = sdg.linear_mx4(x, wc, ws, residual=res) if plain else sdg.linear_mx4(xc, wc, ws, residual=res, xscale=xs)
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    guard = torch.full((M + 2, N), 7.0, dtype=torch.float16, device=cuda)
    P = sdg._ptr
    torch.cuda.synchronize()
    code = sdg.lib().sdg_selftest_stalled_linear_mx4(
        P(x) if plain else P(xc), None if plain else P(xs), M, K, P(wc), P(ws), N, P(res), P(guard[1:]), f, who, stall, 1000,
        P(err), None)
    msg = sdg.last_error()
    assert code == SDG_ERR_DEVICE and any(c in msg for c in ("0x101", "0x102", "0x103")), (code, msg)
    assert int(err) == 0                                        # the call cleared the word it reported
    assert bool((guard[0] == 7).all()) and bool((guard[-1] == 7).all())
    again = sdg.linear_mx4(x, wc, ws, residual=res) if plain else sdg.linear_mx4(xc, wc, ws, residual=res, xscale=xs)
    assert torch.equal(again, want)
    close(again, *linear_ref(op64(xc, xs, K), op64(wc, ws, K), None, res, 0))


def test_stalled_product_that_never_reaches_the_stall(sdg, cuda):
    f, M, N, K, _ = STALLED["narrow"]
    wc, ws = weight(sdg, N, K, 1)
    xc, xs = sdg.quantize_mx4(rnd(M, K, seed=2, dtype=torch.float16))
    y = torch.empty(M, N, dtype=torch.float16, device=cuda)
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    P = sdg._ptr
    assert sdg.lib().sdg_selftest_stalled_linear_mx4(P(xc), P(xs), M, K, P(wc), P(ws), N, None, P(y), f, 0, 1000, 2000000,
                                                     P(err), None) == 0
    assert torch.equal(y, sdg.linear_mx4(xc, wc, ws, xscale=xs))


def test_stalled_product_rejects_bad_arguments(sdg, cuda):
    wc, ws = weight(sdg, 192, 640, 1)
    xc, xs = sdg.quantize_mx4(rnd(1000, 640, seed=2, dtype=torch.float16))
    y = torch.empty(1000, 192, dtype=torch.float16, device=cuda)
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    P = sdg._ptr
    base = {"x": P(xc), "xs": P(xs), "M": 1000, "K": 640, "wc": P(wc), "ws": P(ws), "N": 192, "r": None, "y": P(y), "form": 2,
            "who": 0, "it": 0, "us": 1000, "err": P(err), "st": None}
    call = lambda **k: sdg.lib().sdg_selftest_stalled_linear_mx4(*(base | k).values())
    assert call(form=4) == call(form=0, M=4) == call(who=1) == call(who=2) == call(it=-1) == call(us=0) == call(us=2000001) \
        == call(x=None) == call(xs=None) == 2


def test_status_reports_products_without_a_word(sdg, cuda):
    """A product that had no error word of its own: the failure is reported once, by the next status call."""
    f, M, N, K, _ = STALLED["narrow"]
    wc, ws = weight(sdg, N, K, 1)
    xc, xs = sdg.quantize_mx4(rnd(M, K, seed=2, dtype=torch.float16))
    want = sdg.linear_mx4(xc, wc, ws, xscale=xs)
    y = torch.empty_like(want)
    P = sdg._ptr
    sdg.mx4_status()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    assert sdg.lib().sdg_selftest_stalled_linear_mx4(P(xc), P(xs), M, K, P(wc), P(ws), N, None, P(y), f, 0, 1, 1000, None,
                                                     side.cuda_stream) == 0
    behind = sdg.linear_mx4(xc, wc, ws, xscale=xs, stream=side.cuda_stream)
    side.synchronize()
    assert torch.equal(behind, want)
    with pytest.raises(sdg.SdgError) as ei:
        sdg.mx4_status(stream=side.cuda_stream)
    assert ei.value.code == SDG_ERR_DEVICE and "0x10" in str(ei.value)
    sdg.mx4_status()
    sdg.mx4_status(device=0)


def test_status_refuses_a_captured_stream(sdg, cuda):
    x = torch.zeros(4, device=cuda)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        x += 1
        with pytest.raises(sdg.SdgError) as ei:
            sdg.mx4_status()
    assert ei.value.code == 2
    g.replay()
    torch.cuda.synchronize()
    assert bool((x == 1).all())
