"""8-bit caches whose scales have any sign and size, single and few tokens and prompts, against the formula in 64 bits.

Tolerance, relative to the sum of |weight * value| of a row (A), which is what the signs cannot cancel: scores and sums as in
test_gpu_cache (2e-5); one rounding of the weights to fp16 (bf16 models, few tokens: 2^-11, half a step) or to
the model's type (prompts: u), or two parts (fp16 models, few tokens: 2^-22).  Then the result's own rounding, and in fp16 its
smallest step.  A weight times its scale that lies below 2^-29 of the row's largest is a subnormal fp16 number, off by 2^-40 of that largest and
no more: 2000 of them are 2^-29 of A, which the 2e-5 has room for.
"""
import pytest
import torch

import ksmm_b200 as kb
from test_gpu_cache import DEV, attended, make, unit

pytestmark = pytest.mark.gpu
F8 = torch.float8_e4m3fn


def sizes(cache):
    """The cache with the absolute values of its values."""
    return kb.KVCache.of(cache.keys, (cache.values.view(torch.uint8) & 127).view(F8), cache.key_scales, cache.value_scales.abs())


def close(out, ref, total, rounding):
    t = out.dtype
    most = unit(t) * ref.abs() + (2e-5 + rounding) * total + (2.0 ** -24 if t == torch.float16 else 0)
    off = (out.double() - ref).abs()
    assert (off <= most).all(), (off / most).max().item()


def rounding(dtype, few):
    return (2.0 ** -11 if dtype == torch.bfloat16 else 2.0 ** -22) if few else unit(dtype)


SIGNS = [(-1, -1, -1), (-1, 1, 1), (-1, 0, 1), (0, 0, 0), (0, 0, -1)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads,kv,dim", [(6, 6, 64), (8, 2, 128), (4, 1, 256), (32, 2, 112)])
@pytest.mark.parametrize("new", [1, 2])
def test_signs(new, heads, kv, dim, dtype):
    gen = torch.Generator().manual_seed(dim + new)
    for lengths in ([40, 333, 1, 129], [3000, 64, 700, 5]):  # whole items, and items in parts
        lengths = [max(n, new) for n in lengths]
        cache, table, L, _, q, _, _ = make(gen, lengths, [new] * 4, heads, kv, dim, 16, dtype, eight=True)
        scales = cache.value_scales.clone()
        for signs in SIGNS:
            pick = torch.randint(0, 3, scales.shape, generator=gen)
            cache.value_scales.copy_(scales * torch.tensor(signs, dtype=torch.float32)[pick].to(DEV))
            ref, total = (attended(q, c, table, lengths, [new] * 4) for c in (cache, sizes(cache)))
            close(kb.cache_attention(q, cache, table, L), ref, total, rounding(dtype, True))
    kb.check_device()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads,kv,dim", [(6, 6, 64), (8, 2, 128), (4, 1, 256)])
@pytest.mark.parametrize("new", [1, 3])
def test_sizes(new, heads, kv, dim, dtype):
    """Scales over 24 powers of two in one sequence."""
    gen = torch.Generator().manual_seed(dim + new)
    lengths = [50, 333, 2600]
    cache, table, L, _, q, _, _ = make(gen, lengths, [new] * 3, heads, kv, dim, 16, dtype, eight=True)
    size = torch.exp2(torch.randint(-24, 1, cache.value_scales.shape, generator=gen).float())
    sign = torch.randint(0, 2, size.shape, generator=gen).float() * 2 - 1
    cache.value_scales.mul_((size * sign).to(DEV))
    ref, total = (attended(q, c, table, lengths, [new] * 3) for c in (cache, sizes(cache)))
    close(kb.cache_attention(q, cache, table, L), ref, total, rounding(dtype, True))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("ratio", [2.0 ** 16, 2.0 ** 20])
@pytest.mark.parametrize("first", [False, True])
def test_a_large_scale_of_little_weight(first, ratio, dtype):
    """One token whose values are up to 2^20 times the others' and whose weight is about as small: what the others give is not
    lost.  bf16: 2^20, 40 nats down (its part is 2^-38); fp16: the others' values small, their sum well above the type's smallest."""
    gen = torch.Generator().manual_seed(int(ratio) % 97 + first)
    n, heads, kv, dim = 600, 8, 2, 64
    cache, table, L, _, q, _, _ = make(gen, [n], [1], heads, kv, dim, 16, dtype, eight=True)
    far = 3 if first else n - 2
    page, slot = table[0, far // 16].long(), far % 16
    q[..., 0] = 8.0
    cache.keys.view(torch.uint8)[page, :, slot] = 0
    cache.keys.view(torch.uint8)[page, :, slot, 0] = 0x78  # 256
    cache.key_scales[page, :, slot] = -40.0 / 256  # score: 8 * -40 / sqrt(64) = -40
    cache.value_scales[page, :, slot] *= ratio if dtype == torch.bfloat16 else 1
    if dtype == torch.float16:
        cache.value_scales.div_(ratio / 2.0 ** 7)
        cache.value_scales[page, :, slot] *= ratio
    ref, total = (attended(q, c, table, [n], [1]) for c in (cache, sizes(cache)))
    close(kb.cache_attention(q, cache, table, L), ref, total, rounding(dtype, True))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_few_tokens_and_prompts_agree_with_the_formula(dtype):
    """The same cache with negative scales, as the last 1, 2, 20 and 300 tokens see it."""
    gen = torch.Generator().manual_seed(3)
    n, heads, kv, dim = 333, 8, 2, 64
    cache, table, L, _, q, _, _ = make(gen, [n], [n], heads, kv, dim, 16, dtype, eight=True)
    cache.value_scales.neg_()
    cache.key_scales.mul_(torch.randint(0, 2, cache.key_scales.shape, generator=gen).float().to(DEV) * 2 - 1)
    for last in (1, 2, 20, 300):
        ref, total = (attended(q[-last:], c, table, [n], [last]) for c in (cache, sizes(cache)))
        close(kb.cache_attention(q[-last:], cache, table, L), ref, total, max(rounding(dtype, few) for few in (False, True)))


@pytest.mark.parametrize("sign", [1, -1])
def test_scales_up_to_what_fp16_holds(sign):
    """Small codes with large scales: prompts, single tokens and the formula agree as far as elements lie in the type's range."""
    gen = torch.Generator().manual_seed(7)
    n, heads, kv, dim = 333, 8, 2, 64
    cache, table, L, _, q, _, _ = make(gen, [n], [n], heads, kv, dim, 16, torch.float16, eight=True)
    cache.values.copy_((0.25 * torch.randn(cache.values.shape, generator=gen)).clamp(-0.9, 0.9).to(F8).to(DEV))
    cache.value_scales.copy_(sign * torch.exp2(torch.rand(cache.value_scales.shape, generator=gen) * 15.99))
    for last in (1, 2, 300):
        ref, total = (attended(q[-last:], c, table, [n], [last]) for c in (cache, sizes(cache)))
        close(kb.cache_attention(q[-last:], cache, table, L), ref, total, rounding(torch.float16, last < 20))
