"""Child process of test_gpu_experts_edges.py: runs the checks named on the command line and prints a JSON
line for each. Not collected by pytest.

Oracles are the formulas in 64 bits; U32 is the largest relative error of one float32 rounding."""
import json
import os
import sys
import traceback

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)
from h2o4gpu_amd import codebook4  # noqa: E402

U32 = 2.0 ** -24


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def codebook_of_all_experts():
    """More rows and more values than a fit takes: the second expert's values are in the sample. Its scaled
    values lie in the outer fifth, where a codebook of the first expert's alone has its entries wide apart."""
    first = torch.randn(4000, 320, generator=gen(70))
    second = 0.8 + 0.2 * torch.rand(4000, 320, generator=gen(71))
    second = torch.where(torch.rand(second.shape, generator=gen(72)) < 0.5, -second, second)
    W = torch.stack([first, second]).cuda()

    def error(book):
        q = codebook4.quantize(W[1], 32, book)
        scale = q.scales().repeat_interleave(32, 1)
        return float(((q.dequantize() - W[1]) / scale).square().mean())

    joint = error(codebook4.quantize(W, 32).codebook)
    alone = error(codebook4.quantize(W[0], 32).codebook)
    # sixteen entries of a mixture by halves: a third of the error at most (about an eighth, were they those of
    # Lloyd's fixed point on the whole matrices)
    assert joint < alone / 3, (joint, alone)


def main():
    for name in sys.argv[1:]:
        print("# " + name, flush=True)
        r = dict(name=name, ok=True, why="")
        try:
            globals()[name]()
            torch.cuda.synchronize()
        except Exception as e:  # reported to the collecting test
            r.update(ok=False, why="".join(traceback.format_exception_only(type(e), e))[:1500] +
                     "".join(traceback.format_tb(e.__traceback__)[-2:])[:1000])
            if "HIP error" in r["why"] or "CUDA error" in r["why"]:
                print(json.dumps(r), flush=True)
                return 1  # nothing more is run on the GPU
        print(json.dumps(r), flush=True)
        torch.cuda.empty_cache()
    return 0


if __name__ == "__main__":
    sys.exit(main())
