"""Several host threads make their first calls of the same kernels at a time, each with a batch size, a workspace and a stream of
its own (run as a program of its own: only first calls set a kernel up).  Prints the calls that were refused.

  threads_driver.py scored     attention with modified scores, every instantiation
  threads_driver.py fused      append and attention of a decode step in one launch"""
import ctypes as C
import sys
import threading

import torch

from paged_fixture import load_b200

THREADS, ROWS = 8, 512


def main(what):
    b = load_b200()
    L = b.lib()
    workspaces = [b.Workspace(ROWS) for _ in range(THREADS)]
    streams = [torch.cuda.Stream() for _ in range(THREADS)]
    refused, calls = [], 0
    for dtype in (b.BF16, b.F32):
        for hd in (4, 8, 16, 32, 64, 128, 256):
            for group in GROUPS[what]:
                if dtype == b.BF16 and hd < 8:
                    continue
                ints = lambda n, v: torch.full((n,), v, dtype=torch.int32, device="cuda")
                layer = b.PagedLayer(THREADS * ROWS, 1, hd, dtype, torch.arange(THREADS * ROWS, dtype=torch.int32, device="cuda")[:, None])
                q = torch.zeros(ROWS, group * hd, device="cuda")
                kv = torch.zeros(ROWS, hd, device="cuda")
                outs = [torch.empty(ROWS, group * hd, device="cuda") for _ in range(THREADS)]
                slots = [torch.arange(i * ROWS, (i + 1) * ROWS, dtype=torch.int32, device="cuda") for i in range(THREADS)]
                d_len, d_ring, d_prefill = (ints(THREADS * ROWS, 0) for _ in range(3))
                torch.cuda.synchronize()
                start, score = threading.Barrier(THREADS), b.Score()

                def work(i):
                    torch.cuda.set_device(0)
                    rows = ROWS if i % 2 else 32 + i
                    start.wait()
                    for again in range(3):
                        rc = CALL[what](b, L, layer, score, q, kv, d_len, d_ring, d_prefill, slots[i], rows, group, outs[i], workspaces[i], streams[i])
                        if rc:
                            refused.append((hd, group, dtype, rows, again, L.uocr_b200_last_error().decode()))
                threads = [threading.Thread(target=work, args=(i,)) for i in range(THREADS)]
                for t in threads:
                    t.start()
                for t in threads:
                    t.join()
                torch.cuda.synchronize()
                calls += 3 * THREADS
    assert all(ws.status() == 0 for ws in workspaces)
    print(f"{len(refused)} of {calls} calls refused {refused[:3]}")
    return 1 if refused else 0


def scored(b, L, layer, score, q, kv, d_len, d_ring, d_prefill, slots, rows, group, out, ws, stream):
    return L.uocr_b200_rswa_attention_scored_batch_paged(
        C.byref(layer.desc), C.byref(score.desc), q.data_ptr(), b.F32, d_len.data_ptr(), d_ring.data_ptr(), d_prefill.data_ptr(), slots.data_ptr(), rows, 16,
        group, out.data_ptr(), None, ws.h, stream.cuda_stream)


def fused(b, L, layer, score, q, kv, d_len, d_ring, d_prefill, slots, rows, group, out, ws, stream):
    return L.uocr_b200_rswa_decode_step_paged(
        C.byref(layer.desc), q.data_ptr(), kv.data_ptr(), kv.data_ptr(), d_len.data_ptr(), d_ring.data_ptr(), d_prefill.data_ptr(), slots.data_ptr(), rows, 16,
        group, out.data_ptr(), ws.h, stream.cuda_stream)


CALL = {"scored": scored, "fused": fused}
GROUPS = {"scored": (1, 2, 4), "fused": (1,)}

if __name__ == "__main__":
    sys.exit(main(sys.argv[1]))
