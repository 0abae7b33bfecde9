"""``kernels.dequant_inverse_rotate`` of 4-bit records: it takes the slots that it takes with 2-bit ones."""

import pytest
import torch

from oscar_new_amd import kernels
from tests._int4 import DEV, layout_of, records

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [2, 4])
@pytest.mark.parametrize("dtype", [torch.int64, torch.int32])
@pytest.mark.parametrize("shape", [(12,), (3, 4), (2, 3, 2), (0,)])
def test_slots_of_any_integer_type_and_shape(bits, dtype, shape):
    layout = layout_of(2, bits=bits)
    gen = torch.Generator(device=DEV).manual_seed(5)
    history = torch.zeros(2, layout.stripe_page_bytes, dtype=torch.uint8, device=DEV)
    n = 2 * 768
    if bits == 4:
        history[:, : 768 * 2 * 272] = records(2 * n, gen).view(2, -1)
    else:
        rows = [torch.randn(n, 2, 256, generator=gen, device=DEV).bfloat16() for _ in range(2)]
        kernels.store_int2(*rows, history, torch.arange(n, device=DEV),
                           torch.tensor([1, n], dtype=torch.int32, device=DEV), layout)
    rk, rv = (torch.linalg.qr(torch.randn(256, 256, generator=gen, device=DEV))[0].bfloat16()
              for _ in range(2))
    slots = torch.randint(n, shape, generator=gen, device=DEV, dtype=dtype)
    got = kernels.dequant_inverse_rotate(history, slots, rk, rv, layout)
    values = kernels.read_records(history, slots.long().flatten(), layout)
    for x, value, r in zip(got, values, (rk, rv)):
        assert x.shape == (slots.numel(), 2, 256)
        assert torch.equal(x, kernels.rotate(value, r.T))


@pytest.mark.parametrize("bits", [2, 4])
def test_too_many_slots_are_refused(bits):
    layout = layout_of(1, bits=bits)
    history = torch.zeros(layout.stripe_page_bytes, dtype=torch.uint8, device=DEV)
    r = torch.eye(256, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(ValueError, match="4096"):
        kernels.dequant_inverse_rotate(history, torch.zeros(4097, dtype=torch.int64, device=DEV), r, r, layout)
