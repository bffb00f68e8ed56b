"""Products with 4-bit weights called by several threads of one program."""
import pytest
import torch

from cajeta_llm_b200.csrc import kernels as K
from test_gpu_q4 import DEV, F64, check, sums, weight

pytestmark = pytest.mark.gpu


def test_products_of_several_sizes_from_several_threads_at_once():
    """Tiles of 96 and of 160 rows ask the same kernel for different shared memory: neither call takes the other's away."""
    import threading
    w, full = weight((2048, 64), 64, seed=1)
    failed, go = [], threading.Barrier(8, timeout=60)

    def calls(rows):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                x = torch.randn((rows, 64), device=DEV).to(torch.bfloat16)
                out = torch.empty((rows, 2048), device=DEV)
                go.wait()
                for _ in range(4000):
                    K.gemm_q4(x, w, out)
                torch.cuda.current_stream().synchronize()
                xd = x.to(F64)
                check(out, xd @ full.T, sums(64, xd.abs() @ full.abs().T))
        except Exception as e:
            failed.append((rows, e))

    threads = [threading.Thread(target=calls, args=(rows,)) for rows in (96, 1024) * 4]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed
