"""Low-rank adapters of many requests beside a shared projection.

A packed Linear's weights are shared by every request of a batch; a request
that brings a fine-tune of its own adds  scale * (x D^T) U^T  to its rows, D
[rank, in] and U [out, rank] the two halves of the adapter.  An AdapterBank
keeps the adapters of one Linear on the device, in slots that are loaded and
unloaded while the server runs; low_rank_add applies to each row the adapter
of the slot that the row names, so that one call serves requests of several
adapters, of none, and of one token each (kernels in csrc/low_rank.hip).
fp32 activations as everywhere here, products and sums of fp32 precision;
adapters are kept in fp32, bf16 or fp16.
"""
from __future__ import annotations

from ._lib import enqueue, load_library, no_gradients, rows_of

# the library's limits
MAX_RANK = 512
MAX_SLOTS = MAX_FEATURES = 1 << 20
MAX_ROWS = 1 << 27


def _types(torch):
    return {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _tiled(torch, values, tile):
    """values [S, rows, cols] -> [S, ceil(rows/16), ceil(cols/32), 4, 16, 8], the tiles that the kernels read, zero
    past rows and cols; fp32 as three bf16 planes of each tile, [.., 3, 4, 16, 8], whose sum is the value bit for bit
    (8 bits each, by truncation).  Written to `tile`, or a new tensor."""
    S, rows, cols = (int(s) for s in values.shape)
    r16, c32 = -(-rows // 16), -(-cols // 32)
    if (rows, cols) != (16 * r16, 32 * c32):
        padded = torch.zeros((S, 16 * r16, 32 * c32), dtype=values.dtype, device=values.device)
        padded[:, :rows, :cols] = values
        values = padded
    tiles = values.reshape(S, r16, 16, c32, 4, 8).permute(0, 1, 3, 4, 2, 5)
    if values.dtype != torch.float32:
        return tiles.contiguous() if tile is None else tile.copy_(tiles)
    if tile is None:
        tile = torch.empty((S, r16, c32, 3, 4, 16, 8), dtype=torch.bfloat16, device=values.device)
    left = tiles
    for i in range(3):
        upper = (left.view(torch.int32) & -65536).view(torch.float32)
        tile[:, :, :, i] = upper
        left = left - upper
    return tile


def _sizes_fit(slots, in_features, out_features, max_rank):
    if not (1 <= slots <= MAX_SLOTS and 1 <= in_features <= MAX_FEATURES and 1 <= out_features <= MAX_FEATURES
            and 1 <= max_rank <= MAX_RANK):
        raise ValueError(f"an AdapterBank has 1..{MAX_SLOTS} slots, 1..{MAX_FEATURES} features in and out and a rank of "
                         f"1..{MAX_RANK}")


class AdapterBank:
    """Adapters of one Linear [in_features -> out_features] in `slots` slots of at most max_rank.

    The bank holds its own copies, in `dtype` (fp32, bf16 or fp16; values of another type are rounded to it; fp32 takes
    6 bytes a value: the three bf16 terms that the matrix cores multiply).
    load and unload run on torch's current stream: calls that use the bank on another stream have to be ordered
    after them, and before them when they still read the slot."""

    def __init__(self, slots, in_features, out_features, max_rank, dtype=None, device="cuda"):
        import torch

        dtype = torch.float32 if dtype is None else dtype
        if dtype not in _types(torch):
            raise ValueError("an AdapterBank holds fp32, bf16 or fp16")
        self.slots, self.in_features, self.out_features = int(slots), int(in_features), int(out_features)
        self.max_rank, self.dtype = int(max_rank), dtype
        _sizes_fit(self.slots, self.in_features, self.out_features, self.max_rank)
        k32, n16 = -(-self.in_features // 32), -(-self.out_features // 16)
        tile, held = ((3, 4, 16, 8), torch.bfloat16) if dtype == torch.float32 else ((4, 16, 8), dtype)
        self.down = torch.zeros((self.slots, -(-self.max_rank // 16), k32, *tile), dtype=held, device=device)
        self.up = torch.zeros((self.slots, n16, -(-self.max_rank // 32), *tile), dtype=held, device=device)
        self.scale = torch.zeros(self.slots, dtype=torch.float32, device=device)
        self.rank = torch.zeros(self.slots, dtype=torch.int32, device=device)  # 0: nothing loaded
        self.device, self.index, self.type_id = self.down.device, self.down.get_device(), _types(torch)[dtype]

    def _slot(self, slot):
        if not 0 <= int(slot) < self.slots:
            raise ValueError(f"slot {slot} is outside 0..{self.slots - 1}")
        return int(slot)

    def load(self, slot, down, up, scale=1.0):
        """Puts an adapter into a slot: down [rank, in], up [out, rank], 1 <= rank <= max_rank."""
        import torch

        slot = self._slot(slot)
        if (not torch.is_tensor(down) or not torch.is_tensor(up) or down.dim() != 2 or up.dim() != 2
                or int(down.shape[1]) != self.in_features or int(up.shape[0]) != self.out_features
                or down.shape[0] != up.shape[1]):
            raise ValueError(f"an adapter of this bank is down [rank, {self.in_features}], "
                             f"up [{self.out_features}, rank]")
        rank = int(down.shape[0])
        if not 1 <= rank <= self.max_rank:
            raise ValueError(f"rank {rank} is outside 1..{self.max_rank}")
        with torch.no_grad():
            whole_down = torch.zeros((1, self.max_rank, self.in_features), dtype=self.dtype, device=self.device)
            whole_up = torch.zeros((1, self.out_features, self.max_rank), dtype=self.dtype, device=self.device)
            whole_down[0, :rank] = down
            whole_up[0, :, :rank] = up
            _tiled(torch, whole_down, self.down[slot:slot + 1])
            _tiled(torch, whole_up, self.up[slot:slot + 1])
            self.scale[slot] = float(scale)
            self.rank[slot] = rank
        return slot

    def unload(self, slot):
        """Empties a slot: rows that name it are left as they are without an adapter."""
        self.rank[self._slot(slot)] = 0

    @classmethod
    def stack(cls, down, up, scale, ranks=None):
        """A full bank from stacked adapters: down [slots, R, in], up [slots, out, R] of one type on one device,
        scale [slots]; ranks: how much of R each slot uses (a list; default all), what is past it is not read."""
        import torch

        if (not torch.is_tensor(down) or not torch.is_tensor(up) or down.dim() != 3 or up.dim() != 3
                or down.shape[0] != up.shape[0] or down.shape[1] != up.shape[2] or down.dtype != up.dtype
                or down.device != up.device):
            raise ValueError("stacked adapters are down [slots, R, in] and up [slots, out, R] of one type and device")
        S, R, K = (int(s) for s in down.shape)
        ranks = [R] * S if ranks is None else [int(r) for r in ranks]
        if len(ranks) != S or any(not 0 <= r <= R for r in ranks):
            raise ValueError(f"ranks are {S} numbers of 0..{R}")
        scale = torch.as_tensor(scale, dtype=torch.float32, device=down.device)
        if tuple(scale.shape) != (S,):
            raise ValueError(f"scale must be [{S}]")
        bank = cls.__new__(cls)
        if down.dtype not in _types(torch):
            raise ValueError("an AdapterBank holds fp32, bf16 or fp16")
        _sizes_fit(S, K, int(up.shape[1]), R)
        bank.slots, bank.in_features, bank.out_features, bank.max_rank = S, K, int(up.shape[1]), R
        bank.dtype, bank.device, bank.index = down.dtype, down.device, down.get_device()
        bank.type_id = _types(torch)[down.dtype]
        with torch.no_grad():
            bank.rank = torch.tensor(ranks, dtype=torch.int32, device=down.device)
            bank.scale = scale.clone()
            if min(ranks) < R:
                live = torch.arange(R, device=down.device) < bank.rank[:, None]
                zero = torch.zeros((), dtype=down.dtype, device=down.device)
                down, up = torch.where(live[:, :, None], down, zero), torch.where(live[:, None, :], up, zero)
            bank.down, bank.up = _tiled(torch, down, None), _tiled(torch, up, None)
        return bank


def adapter_rows(lengths, slots, device="cuda"):
    """The slot of each row, int32, of requests of these lengths in a row: slots[i] for the rows of request i, -1
    for a request without an adapter."""
    import torch

    if len(lengths) != len(slots) or any(int(n) < 0 for n in lengths):
        raise ValueError("adapter_rows takes one slot and one length for each request")
    slots = torch.tensor([int(s) for s in slots], dtype=torch.int32)
    return slots.repeat_interleave(torch.tensor([int(n) for n in lengths], dtype=torch.int64)).to(device)


def low_rank_add(y, x, bank, rows, *, out=None, library=None):
    """out = y + each row's adapter of x:  y[m] + scale[a] (x[m] down[a]^T) up[a]^T,  a = rows[m].

    y [..., out] is the shared projection of x [..., in], both fp32 on the GPU with unit column stride and one row
    stride (column ranges of wider rows pass); rows [M] int32, contiguous.  A row whose number is no loaded slot of
    the bank (negative, out of range, unloaded) keeps y.  out: None for a new tensor, y itself (rows without an
    adapter are not touched), or another that overlaps nothing that is read.  A row of x that holds an infinity or NaN
    gives NaN; other rows are not affected.  fp32 factors below 2^-110 count in steps of 2^-133.  Runs on torch's
    current stream; capturable into a HIP graph.  No gradients."""
    import torch

    if not isinstance(bank, AdapterBank):
        raise ValueError("low_rank_add needs an AdapterBank")
    M, y_stride = rows_of(torch, "y", y, bank.out_features)
    Mx, x_stride = rows_of(torch, "x", x, bank.in_features)
    no_gradients(torch, y, x, out)
    if Mx != M or M > MAX_ROWS:
        raise ValueError(f"y has {M} rows, x has {Mx}: as many of both are wanted, at most {MAX_ROWS}")
    if not (isinstance(rows, torch.Tensor) and rows.dtype == torch.int32 and rows.numel() == M
            and rows.is_contiguous()):
        raise ValueError(f"rows must be a contiguous int32 tensor of {M} slots")
    at = y.get_device()
    if out is None:
        out_stride = bank.out_features  # (rows at that stride are contiguous)
        out = torch.empty_like(y) if y_stride == out_stride else y.new_empty(y.shape)
    elif out is y:
        out_stride = y_stride
    else:
        Mo, out_stride = rows_of(torch, "out", out, bank.out_features)
        if Mo != M:
            raise ValueError(f"out has {Mo} rows, y has {M}")
    if not at == x.get_device() == rows.get_device() == out.get_device() == bank.index:
        raise ValueError("y, x, rows, out and the bank must be on one GPU")
    if M == 0:
        return out
    lib = load_library(library)
    sizes = (M, bank.in_features, bank.out_features, bank.slots, bank.max_rank, bank.type_id)
    need = lib.tsplat_low_rank_scratch_bytes(*sizes)
    scratch = torch.empty(need, dtype=torch.uint8, device=y.device) if need else None
    enqueue(lib, "tsplat_low_rank_add_async", at, y.data_ptr(), y_stride, x.data_ptr(), x_stride, rows.data_ptr(),
            bank.down.data_ptr(), bank.up.data_ptr(), bank.scale.data_ptr(), bank.rank.data_ptr(), out.data_ptr(),
            out_stride, *sizes, scratch.data_ptr() if need else None, need)
    return out
