"""What a kernel context holds: contexts that never see a paged cache (a decoder's
net and its argmax) take no room for one, and a context's products and its paged
attention share their scratch without reaching each other.
"""

import numpy as np
import pytest

from helpers import ensure_library
from test_gpu_paged import Case, attend
from whispereacp_amd import synthetic as S

pytestmark = pytest.mark.gpu

MB = 1 << 20
SMALL = S.DecoderShape(64, 1, 1, 256, 64, 16, 16)


def taken(make):
    """What `make` returns and the device memory it took."""
    import gc
    import torch
    gc.collect()
    torch.cuda.synchronize()
    before = torch.cuda.mem_get_info()[0]
    made = make()
    torch.cuda.synchronize()
    return made, before - torch.cuda.mem_get_info()[0]


def test_a_decoder_takes_its_products_scratch_alone():
    # Two contexts (the net's and the argmax's) of 16 MB each at this shape, and little
    # else; 64 MB more each with room for a paged cache's partial rows.
    ensure_library()
    from whispereacp_amd.decoder import Decoder
    decoder_file = S.synthetic_decoder_file(SMALL, "F32")
    first = Decoder(SMALL, decoder_file)  # (what the library takes once)
    second, more = taken(lambda: Decoder(SMALL, decoder_file))
    assert more < 64 * MB, more / MB
    first.close()
    second.close()


def test_a_kernel_context_holds_one_scratch():
    ensure_library()
    from whispereacp_amd.decoder import KernelContext
    first = KernelContext(SMALL)
    _, more = taken(lambda: KernelContext(SMALL))
    assert more < 80 * MB, more / MB
    assert first.handle


def test_products_and_paged_attention_take_turns_in_the_scratch():
    ensure_library()
    import torch
    from whispereacp_amd.decoder import KernelContext
    from whispereacp_amd import _native as N
    ctx = KernelContext(SMALL)
    case = Case("F16", [2, 1], [3000, 700], 4, 2, 64, 64, seed=3)  # (its keys are split)
    cache, rows = case.cache(), case.packed()
    generator = torch.Generator(device="cuda")
    generator.manual_seed(5)
    x = torch.randn((600, 1280), generator=generator, device="cuda")
    w = torch.randn((1280, 1280), generator=generator, device="cuda").half()
    y = torch.zeros((600, 1280), device="cuda")

    def product():
        y.zero_()
        ctx.linear(x, 600, 1280, w, N.WSP_F16, None, y, 1280, 0)
        torch.cuda.synchronize()
        return y.clone()

    product_alone, attention_alone = product(), attend(ctx, case, cache=cache, rows=rows)
    # 1280 products and sums of fp32, and x's two 16-bit parts.
    exact = x.double().cpu() @ w.double().cpu().T
    bound = x.double().cpu().abs() @ w.double().cpu().abs().T * (1288 * 2.0 ** -24 + 2.0 ** -22)
    assert bool(((product_alone.double().cpu() - exact).abs() <= bound).all())
    for _ in range(3):
        assert np.array_equal(attend(ctx, case, cache=cache, rows=rows), attention_alone)
        assert torch.equal(product(), product_alone)
