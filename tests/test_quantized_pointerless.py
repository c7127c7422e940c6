"""torch.vmap's tensors, which have no memory of their own, given to the torch functions: every call raises with the
interpreter's lock held, before it does anything on the device. The tensors are fake ones that say they are on a GPU: none is
needed, so this runs anywhere."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

BF, I8, I32, F32, U8 = torch.bfloat16, torch.int8, torch.int32, torch.float32, torch.uint8


def _empty(dtype, *shape):
    return torch.empty(shape, dtype=dtype, device="cuda")


def _cache():
    return (_empty(U8, 4, 2, 16, 64), _empty(U8, 4, 2, 64, 16), _empty(BF, 4, 2, 16, 2), _empty(BF, 4, 2, 16, 2))


# arguments of a call; every one in turn is the slice of a batch
CALLS = {
    "rms_norm_quant": lambda: [_empty(BF, 5, 96), _empty(BF, 96), _empty(BF, 5, 96)],
    "linear_int8": lambda: [_empty(I8, 5, 96), _empty(I8, 8, 96), _empty(F32, 5), _empty(F32, 8), _empty(F32, 8)],
    "reshape_and_cache_int4": lambda: [_empty(BF, 5, 2, 128), _empty(BF, 5, 2, 128), *_cache(), _empty(I32, 5)],
    "paged_cache_load_int4": lambda: [*_cache(), _empty(I32, 2, 3), _empty(I32, 2), 10, _empty(I32, 2)],
    "paged_attention_int4": lambda: [_empty(BF, 2, 4, 128), *_cache(), _empty(I32, 2, 3), _empty(I32, 2), 0.1],
}


@pytest.mark.parametrize("name", CALLS)
def test_batched_tensors_raise(pkg, name):
    with FakeTensorMode():
        args = CALLS[name]()
        more = dict(out_dtype=BF) if name == "linear_int8" else {}
        for i in (i for i, t in enumerate(args) if isinstance(t, torch.Tensor)):
            batch = args[i].unsqueeze(0).expand(3, *args[i].shape).clone()
            with pytest.raises(RuntimeError, match="data pointer"):
                torch.vmap(lambda t: getattr(pkg.quantized, name)(*args[:i], t, *args[i + 1:], **more))(batch)
