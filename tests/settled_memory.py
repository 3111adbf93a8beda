"""Memory that stays for longer than a test: the workspaces that torch's libraries take with a thread's first product, and keep.  Cut from a large block that a test has left in the cache they
would keep all of it from going back to the device, and tests of little memory behind would find other room than they measure."""
import gc

import torch


def settle():
    """Frees what is cached, and has the libraries take their workspaces, of this thread and of autograd's, from the device."""
    gc.collect()
    torch.cuda.empty_cache()
    for dtype in (torch.float32, torch.float64, torch.float16, torch.bfloat16):
        a, b = (torch.ones((64, 64), device="cuda", dtype=dtype, requires_grad=True) for _ in range(2))
        torch.autograd.grad((a @ b).sum(), (a, b))
    del a, b
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
