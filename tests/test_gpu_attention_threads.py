"""First calls of the serving attention kernels from several host threads at
once, through the C ABI (which runs without Python's lock), each on a stream
and a workspace of its own."""
import ctypes
import math
import threading

import pytest
import torch

import cabi
from seq_reference import U, attend, check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,code", [(torch.float16, cabi.F16), (torch.bfloat16, cabi.BF16)])
@pytest.mark.parametrize("path", [cabi.PATH_TC, cabi.PATH_SKINNY, cabi.PATH_SIMT])
@pytest.mark.parametrize("d", [64, 128])
def test_threads(cuda, dtype, code, path, d):
    n, hq, hkv, threads = 200, 8, 2, 6
    g = torch.Generator(device="cuda").manual_seed(d)
    q = torch.randn(threads, n, hq, d, generator=g, device="cuda").to(dtype)
    k, v = (torch.randn(n, hkv, d, generator=g, device="cuda").to(dtype) for _ in range(2))
    out = torch.empty_like(q)
    cu = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    calls, keep, status = [], [], [None] * threads
    for i in range(threads):
        a = cabi.AttentionSeqArgs()
        a.dtype = a.kv_dtype = code
        a.Q, a.K, a.V, a.O = q[i].data_ptr(), k.data_ptr(), v.data_ptr(), out[i].data_ptr()
        a.batch, a.tokens_q, a.heads_q, a.heads_kv, a.head_dim, a.tokens_kv = 1, n, hq, hkv, d, n
        a.q_stride_token = a.o_stride_token = hq * d
        a.q_stride_head = a.o_stride_head = a.k_stride_head = a.v_stride_head = d
        a.k_stride_row = a.v_stride_row = hkv * d
        a.cu_seqlens_q, a.scale, a.causal, a.path = cu.data_ptr(), 1 / math.sqrt(d), 1, path
        need = cabi.lib().cmpx_attention_seq_workspace_size(ctypes.byref(a))
        ws = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")
        a.workspace, a.workspace_bytes = ws.data_ptr(), need
        keep.append(ws)
        calls.append((a, torch.cuda.Stream()))
    torch.cuda.synchronize()
    gate = threading.Barrier(threads)

    def work(i):
        torch.cuda.set_device(0)
        gate.wait()
        a, s = calls[i]
        status[i] = [cabi.lib().cmpx_attention_seq(ctypes.byref(a), ctypes.c_void_p(s.cuda_stream)) for _ in range(5)]

    pool = [threading.Thread(target=work, args=(i,)) for i in range(threads)]
    for t in pool:
        t.start()
    for t in pool:
        t.join()
    torch.cuda.synchronize()
    assert cabi.device_error() == 0
    assert status == [[cabi.OK] * 5] * threads
    for i in range(threads):
        want, tol = attend(q[i], k, v, 1 / math.sqrt(d), True, U[dtype], U[dtype])
        check(out[i], want, tol, f"thread {i}")
