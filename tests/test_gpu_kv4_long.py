"""GPU tests of jules_hip_kv4_attention over texts so long that what its sums carry
beside the output would show: 65536 to 262144 keys taken by one wave.  The root mean
square error of the output against softmax in 64 bits, on the device."""
import math

import pytest
import torch

from jules_amd import ops
from tests.decoder64 import BF16, F32
from tests.helpers import case

pytestmark = pytest.mark.gpu

i32 = torch.int32


@pytest.mark.parametrize("D,group,new,length", [
    (128, 4, 40, 131072),     # waves of their own rows: a wave has all keys
    (64, 4, 40, 65536), (64, 4, 40, 262144),
    (128, 8, 1, 524288),      # one tile of rows: a wave has every fourth 32 keys
    (64, 8, 5, 300000), (128, 8, 3, 262144), (64, 8, 8, 262144)])
def test_long_texts(dev, D, group, new, length):
    """Flat and sharp softmaxes (q of 1 and of 4 times unit variance).  max_len = 1
    keeps the keys whole.

    The roundings are to nearest and those of different keys independent, so their
    variances add, each a third of the square of the half step at most:
    - the output's, 2^-8 of it;
    - the probabilities' times the value's scale, 2^-8 of what each weighs: the
      code's distance from the middle of the row's range;
    - the scores', as attention64 bounds each: twice that of what each weighs;
    - the sums': products of 32 keys are added with at most 4 roundings of 2^-24 of
      the sum, which holds C = 1 + c/128 (below 2) of at most 1024 keys before the
      middle is taken out of it, and is multiplied by 128 at the end; the same for
      the sum of the probabilities, which is multiplied by the middle of C."""
    page = 256
    g = torch.Generator(dev).manual_seed(length + D)
    pages = -(-length // page)
    cache = ops.KV4Cache.empty(pages, 1, D, page, dev)
    table = torch.arange(pages, dtype=i32, device=dev).view(1, -1)
    lens = torch.tensor([length], dtype=i32, device=dev)
    k, v = torch.randn(2, length, 1, D, generator=g, device=dev)
    ops.kv4_append(cache, k, v, table, lens)
    k, v = (t[:, 0].double() for t in ops.kv4_read(cache, table, lens, length, dtype=torch.float32))
    meta = [m[:, 0].reshape(-1, 2)[:length].double() for m in (cache.k_meta, cache.v_meta)]
    step = meta[1][:, :1]
    far = v - (meta[1][:, 1:] + 7.5 * step)
    key = torch.arange(length, device=dev)
    for size in (1.0, 4.0):
        case(f"kv4 attention D={D} group={group} new={new} length={length} q times {size}")
        q = (size * torch.randn(new, group, D, generator=g, device=dev)).to(torch.bfloat16)
        scale = 1.0 / math.sqrt(D)
        o = ops.kv4_attention(q, cache, table, lens, max_len=1, scale=scale).double().flatten(0, 1)
        torch.cuda.synchronize()
        rows = q.double().flatten(0, 1)
        p = scale * torch.matmul(rows, k.t().contiguous())
        top = p.abs().max()
        last = length - new + torch.arange(new, device=dev).repeat_interleave(group)
        p.masked_fill_(key > last[:, None], -math.inf)
        p = torch.softmax(p, -1)
        want = torch.matmul(p, v)
        err = ((D / 8 + 8) * F32 * scale * 3 * rows.abs().sum(-1).max()
               * (16 * meta[0][:, 0] + meta[0][:, 1].abs()).max() + 8 * F32 * top)
        # of the 1024 keys of a wave's 32 steps; up to 64 rows four waves take steps in turn
        waves = 4 if new * group <= 64 else 1
        held = torch.nn.functional.pad(p * step[:, 0], (0, -length % (1024 * waves)))
        held = held.unflatten(-1, (-1, 32, waves, 32)).sum((-1, -3)).flatten(1).amax(-1)
        sums = 128 * F32 * 2 * held
        var = (BF16 * want).square() + BF16**2 * torch.matmul(p.square(), far.square())
        var = var + (2 * err)**2 * torch.matmul(p.square(), v.square())
        var = var / 3 + (2 * 4 * (length / 32) * sums.square() / 3)[:, None]
        rms = (o - want).square().mean().sqrt().item()
        bound = 1.1 * var.mean().sqrt().item()
        print(f"error {rms / want.square().mean().sqrt().item():.5f} of the output, bound "
              f"{bound / want.square().mean().sqrt().item():.5f}", flush=True)
        assert rms <= bound
