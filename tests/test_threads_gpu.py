"""The library's first call in a thread that has made no CUDA call before."""

from __future__ import annotations

import threading

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"


@pytest.fixture(scope="module", autouse=True)
def _need_cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import flashattntile_b200  # noqa: F401


def _calls():
    import flashattntile_b200 as fat
    from flashattntile_b200.kernels.decode import launch_decode
    from flashattntile_b200.kernels.prefill import launch_prefill

    gen = torch.Generator(device=DEV).manual_seed(1)
    k, v = (torch.randn((12, 16, 2, 64), generator=gen, device=DEV).half() for _ in range(2))
    table = torch.tensor([[3, 4, 5, 0], [3, 4, 6, 0], [3, 4, 7, 8]], dtype=torch.int32, device=DEV)
    cache = fat.PagedKVCache(k, v, table, torch.tensor([40, 33, 60], dtype=torch.int32, device=DEV), 16)
    q = torch.randn((3, 8, 64), generator=gen, device=DEV).half()
    cu = torch.tensor([0, 3], dtype=torch.int32, device=DEV)
    shared = fat.find_shared_prefix(cache, [3])
    out = torch.empty_like(q)
    return {
        "shared_prefix_decode": lambda: fat.shared_prefix_decode_attention(q, cache, shared, out=out),
        "decode": lambda: launch_decode(q, k, v, table, cache.seq_lens, 16, 0.125, out=out),
        "prefill": lambda: launch_prefill(q, q[:, :2], q[:, 2:4], cu, cu, 3, 3, True, 0.125, out=out),
    }


@pytest.mark.parametrize("name", ["shared_prefix_decode", "decode", "prefill"])
def test_first_call_in_a_thread(name):
    import flashattntile_b200 as fat

    call = _calls()[name]
    with fat.value_checks(False):
        want = call().clone()
        got, errors = [], []

        def run():
            try:
                with fat.value_checks(False):
                    got.append(call())
            except Exception as error:  # noqa: BLE001
                errors.append(error)

        thread = threading.Thread(target=run)
        thread.start()
        thread.join()
    assert not errors, errors
    assert torch.equal(got[0], want)
