"""Times of the trainable layers beside torch's: rates of the card, whole networks forward and backward, shapes that perf/operators.py does not list, a lookup gradient's worst tokens.
Usage: python scratch/layer_times.py [rates] [networks] [shapes] [lookup]"""
import os
import sys
import time

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path[:0] = [ROOT, os.path.join(ROOT, "tests")]
import _pkg  # noqa: E402

_pkg.load()
from ibl_nerf_amd import checkpoint as ck, layers as L, model as M  # noqa: E402
from torch_ref import RefShaped  # noqa: E402


def ms(f, n=10):
    """milliseconds a call, the median of three runs of n calls in a row"""
    runs = []
    for _ in range(3):
        f()
        torch.cuda.synchronize()
        t = time.perf_counter()
        for _ in range(n):
            f()
        torch.cuda.synchronize()
        runs.append((time.perf_counter() - t) / n * 1e3)
    return sorted(runs)[1]


def rates():
    for gib in (1, 2, 8):
        x = torch.empty(gib << 30, dtype=torch.uint8, device="cuda")
        y = torch.empty_like(x)
        print("copy of %d GiB: %.0f GB/s" % (gib, 2 * x.numel() / ms(lambda: y.copy_(x)) / 1e6), flush=True)
    n = 8192
    for t in (torch.bfloat16, torch.float16, torch.float32):
        a, b = torch.randn(n, n, device="cuda").to(t), torch.randn(n, n, device="cuda").to(t)
        print("product %d^3 %s: %.0f TFLOP/s" % (n, t, 2 * n ** 3 / ms(lambda: a @ b) / 1e9), flush=True)


def networks():
    for arch in ((8, 512, 10, 4), (10, 384, 12, 5)):
        net = RefShaped(ck.synthetic_arch_state_dict(1, arch), arch).cuda()
        params = list(net.parameters())
        for n, s in ((64, 64), (1024, 64), (4096, 192)):
            pts, d, up = torch.rand(n, s, 3, device="cuda"), torch.randn(n, 3, device="cuda"), torch.randn(n, s, 18, device="cuda")
            for t in (torch.float32, torch.bfloat16):
                def ours():
                    torch.autograd.grad(M.fused_network_query(pts, d, net, layer_dtype=t), params, up)

                def theirs():
                    with torch.autocast("cuda", dtype=t, enabled=t != torch.float32):
                        raw = net(L.encode(pts.reshape(-1, 3), arch[2]), L.encode(d, arch[3]).repeat_interleave(s, 0))
                    torch.autograd.grad(raw.float(), params, up.reshape(-1, 18))
                for who, f in (("layers", ours), ("torch", theirs)):
                    torch.cuda.reset_peak_memory_stats()
                    base = torch.cuda.memory_allocated()
                    took = ms(f, 3)
                    print("IBLNeRF%s %d x %d rays %s %s: %.2f ms, %.2f GiB" % (arch[:2], n, s, t, who, took, (torch.cuda.max_memory_allocated() - base) / 2 ** 30), flush=True)


def shapes():
    def dense(n, k, o, t, keep=True):
        x, w, b = torch.randn(n, k, device="cuda").relu().to(t), (torch.randn(o, k, device="cuda") / k ** 0.5).to(t), torch.randn(o, device="cuda").to(t)
        y, ky = L.dense_forward(x, w, b, relu=True)
        kx, dy = L.checkpoint(x, signed=False), torch.randn(n, o, device="cuda").to(t)
        f = ms(lambda: L.dense_forward(x, w, b, relu=True, keep=keep), 20)
        dx = ms(lambda: L.dense_backward(dy, kx, w, relu=ky, need_dw=False, need_db=False), 20)
        dw = ms(lambda: L.dense_backward(dy, kx, w, relu=ky, need_dx=False), 20)
        ft = ms(lambda: torch.nn.functional.linear(x, w, b), 20)
        print("%d x %d -> %d %s: forward %.1f us%s, dX %.1f, dW %.1f (a library's product %.1f)" % (n, k, o, str(t)[6:], f * 1e3, "" if keep else " (no checkpoint)", dx * 1e3, dw * 1e3, ft * 1e3), flush=True)
    for n in (4096, 8192, 16384, 32767, 32768, 65536):
        dense(n, 512, 512, torch.bfloat16)
    for o in (256, 512, 1024, 1536, 1537, 2048, 2049):
        dense(65536, 512, o, torch.bfloat16)
    for o in (1, 3, 18):
        dense(786432, 512, o, torch.float32, keep=False)
        dense(786432, 512, o, torch.bfloat16, keep=False)
    for r in (352, 368, 512, 528):
        dense(262144, r, 32, torch.bfloat16)


def lookup():
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    for n, d in ((4096, 48), (16384, 16), (16384, 128), (640000, 64)):
        dout = torch.randn(n, d, generator=g, device="cuda")
        for what, index in (("anywhere", torch.randint(0, 65536, (n,), generator=g, device="cuda")), ("on neighbours", torch.randint(0, 256, (n,), generator=g, device="cuda")),
                            ("on multiples of 256", 256 * torch.randint(0, 256, (n,), generator=g, device="cuda"))):
            plain = torch.zeros(65536, d, device="cuda")
            print("lookup gradient of %d x %d, 65 536 tokens, positions %s: %.1f us (index_add_ with its clearing %.1f)"
                  % (n, d, what, ms(lambda: L.lookup_backward(dout, index, 65536), 20) * 1e3, ms(lambda: plain.zero_().index_add_(0, index, dout), 20) * 1e3), flush=True)


if __name__ == "__main__":
    for name in sys.argv[1:] or ["rates", "networks", "shapes", "lookup"]:
        globals()[name]()
