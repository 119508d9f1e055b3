"""GPU: the waits of the rank-side products are bounded, and one that runs out is reported (nothing faults, traps or hangs: a test entry
holds the loads back and gives the waits a short limit)."""
import ctypes as C

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m,c,r", [(700, 1024, 8), (64, 128, 16), (5000, 4096, 3)])
def test_a_wait_that_runs_out_is_reported(cuda, m, c, r):
    from b2g import _lib, ops

    g = torch.Generator(device=cuda).manual_seed(m)
    x = torch.randn(m, c, generator=g, device=cuda).bfloat16()
    w = torch.randn(r, c, generator=g, device=cuda).bfloat16()
    s = torch.randn(m, 16, generator=g, device=cuda).bfloat16()
    p = lambda t: C.c_void_p(t.data_ptr())                                   # noqa: E731
    stream = C.c_void_p(torch.cuda.current_stream().cuda_stream)
    down, grad = ops.lora_down(x, w, False, 2.0, r)[0], ops.lora_wgrad(s, x, 1.0, r, False)
    ops.check_status()
    status = ops.status_word(cuda)
    out = torch.empty(m, 16, dtype=torch.bfloat16, device=cuda)
    _lib.call("b2g_debug_stalled_lora_down", p(x), p(w), p(out), m, c, r, stream)
    torch.cuda.synchronize()
    assert int(status.item()) == 602
    with pytest.raises(_lib.B2GError, match="bounded wait"):
        ops.check_status()
    nbytes = _lib.query("b2g_lora_wgrad_workspace_bytes", m, c)
    ws = torch.zeros(nbytes // 4, device=cuda)
    dw = torch.empty(r, c, dtype=torch.bfloat16, device=cuda)
    _lib.call("b2g_debug_stalled_lora_wgrad", p(s), p(x), p(dw), p(ws), nbytes, m, c, r, stream)
    torch.cuda.synchronize()
    assert int(status.item()) == 612
    with pytest.raises(_lib.B2GError, match="bounded wait"):
        ops.check_status()
    # the next calls are not affected
    assert torch.equal(ops.lora_down(x, w, False, 2.0, r)[0], down) and torch.equal(ops.lora_wgrad(s, x, 1.0, r, False), grad)
    ops.check_status()


def test_the_word_that_these_products_report_to(cuda):
    """Their entries take no status: it is the library's, which check_status reads."""
    from b2g import _lib, ops

    word = C.c_void_p()
    _lib.call("b2g_status_word", C.byref(word))
    assert word.value == ops.status_word(cuda).data_ptr()
