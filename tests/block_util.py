"""What the tests of a block's operators share: a store of given weights, dropout's generator on the
host, and the units of the tolerances."""
import numpy as np

U = 2.0 ** -24  # half a step of fp32, relative


def unit(dtype):
    """Half a step of a type, relative."""
    import torch
    return torch.finfo(dtype).eps / 2


def store_of(weights, mode):
    """A store of `weights` (float tensors; bfloat16-representable where the mode is not fp32)
    between two others, on torch's stream: tensor k of the list is tensor k + 1 of the store."""
    import torch
    import ttperf
    s = ttperf.ParamStore([(100,), *[tuple(w.shape) for w in weights], (70,)], mode=mode)
    s.set_stream(torch.cuda.current_stream())
    for k, w in enumerate(weights):
        if mode == "bf16":
            s.upload(ttperf.BUF_PARAM, k + 1, w.bfloat16().reshape(-1).cuda())
        else:
            s.upload(ttperf.BUF_MASTER, k + 1, w.float().reshape(-1).cuda())
    return s


def param_dtype(mode):
    import torch
    return torch.float32 if mode == "fp32" else torch.bfloat16


def grad(store, k):
    import ttperf
    return store.tensors[k].torch_view(ttperf.BUF_GRAD)


def untouched(store, written, value):
    """Whether the gradients outside the tensors `written` (their padding too) are all `value`."""
    import torch
    import ttperf
    flat = store.torch_view(ttperf.BUF_GRAD)
    mask = torch.ones(store.total, dtype=torch.bool, device="cuda")
    for i in written:
        mask[store.offsets[i]:store.offsets[i] + store.tensors[i].numel] = False
    return bool((flat[mask] == value).all())


def pitched(x, left, right, fill=0.0):
    """x as columns of a wider matrix (a view)."""
    import torch
    wide = torch.full((x.shape[0], left + x.shape[1] + right), fill, dtype=x.dtype, device=x.device)
    view = wide[:, left:left + x.shape[1]]
    view.copy_(x)
    return view


def philox(key, counter):
    """Philox 4x32-10 (Salmon et al., 2011) of 32-bit words: (k0, k1), arrays (c0, c1, c2, c3)."""
    c = [np.asarray(v, np.uint64) for v in counter]
    k = [int(v) for v in key]
    low, sh = np.uint64(0xFFFFFFFF), np.uint64(32)
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> sh) ^ c[1] ^ np.uint64(k[0]), b & low, (a >> sh) ^ c[3] ^ np.uint64(k[1]),
             a & low]
        k = [(k[0] + 0x9E3779B9) % 2 ** 32, (k[1] + 0xBB67AE85) % 2 ** 32]
    return c


def threshold(p):
    return min(round(p * 65536), 65535)


def kept(rows, cols, p, seed, stream, row0=0):
    """Which elements of rows row0 to row0 + rows dropout keeps."""
    groups = -(-cols // 8)
    g = np.arange(row0 * groups, (row0 + rows) * groups, dtype=np.uint64)
    seed, mask = seed % 2 ** 64, 2 ** 32 - 1
    words = philox((seed & mask, seed >> 32),
                   (g & np.uint64(mask), g >> np.uint64(32),
                    np.full_like(g, stream & mask), np.full_like(g, stream >> 32)))
    halves = np.stack([h for w in words for h in (w & np.uint64(0xFFFF), w >> np.uint64(16))], 1)
    return halves.reshape(rows, groups * 8)[:, :cols] >= threshold(p)


def dropped(v, p, seed, stream, residual=None):
    """dropout of a float32 tensor on the host, rounded as the operator's formula rounds."""
    import torch
    keep = torch.from_numpy(kept(v.shape[0], v.shape[1], p, seed, stream))
    t = threshold(p)
    out = v * torch.tensor(65536.0 / (65536.0 - t), dtype=v.dtype)
    if residual is None:
        return torch.where(keep, out, torch.zeros_like(out))
    return torch.where(keep, residual + out, residual)
