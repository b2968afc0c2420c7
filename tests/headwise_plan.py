"""Which kernel a head-wise call runs through: the library's rules for chunks, lanes, heads
an item and blocks, restated for contiguous arrays, so that a test can say which code its
sizes reach."""
import torch

ITEM = {"float32": 4, "float16": 2, "bfloat16": 2}
SHAPES = {8: (1, 2), 4: (1, 4), 2: (1, 4), 1: (1, 4, 16)}           # units a lane, by items a chunk
THREADS = 128
BLOCKS_AN_SM = 4                                                    # of the gradient's kernel, at least
STEPS_AHEAD = 3                                                     # heads an item that its copies ahead need


def _ceil(a, b):
    return -(-a // b)


class Plan:
    """heads, dims: of the call's arrays; rotated: items of each that are rotated."""

    def __init__(self, dtype, tokens, heads, dims, rotated, interleaved, backward=False):
        rotated = [r if r else 0 for r in rotated]
        self.vec = min(self._widest(ITEM[dtype], d, r, interleaved) for d, r in zip(dims, rotated))
        units = max(self._units(d, r, interleaved, self.vec) for d, r in zip(dims, rotated))
        self.lanes = 1
        while self.lanes < 32 and self.lanes < units:
            self.lanes *= 2
        self.iter = min(i for i in SHAPES[self.vec] if i * self.lanes >= units)
        most, busy = (8, 1024) if backward else (16, 512)
        sms = torch.cuda.get_device_properties(0).multi_processor_count
        while most > 1 and tokens * sum(heads) * self.lanes // most < busy * sms:
            most //= 2
        items = [_ceil(h, most) for h in heads]
        self.heads_an_item = [_ceil(h, n) for h, n in zip(heads, items)]
        self.ahead = backward and self.vec * ITEM[dtype] == 16 and self.iter == 1 and min(self.heads_an_item) >= STEPS_AHEAD
        blocks = sum(_ceil(tokens * n, THREADS // self.lanes) for n in items)
        self.rounds = _ceil(blocks, sms * BLOCKS_AN_SM) + 1           # the roles' shares are rounded up
        self.blocks = min(blocks, sms * 8)

    @classmethod
    def launches(cls, dtype, tokens, heads, dims, rotated, interleaved):
        """Plans of a forward call's launches: from 2^20 items on, arrays of different chunks have one each."""
        widths = [cls._widest(ITEM[dtype], d, r or 0, interleaved) for d, r in zip(dims, rotated)]
        if len(set(widths)) == 1 or tokens * sum(h * d for h, d in zip(heads, dims)) < 2 ** 20:
            return [cls(dtype, tokens, heads, dims, rotated, interleaved)]
        return [cls(dtype, tokens, *zip(*[a for a, v in zip(zip(heads, dims, rotated), widths) if v == width]), interleaved)
                for width in sorted(set(widths))]

    @staticmethod
    def _units(dim, rot, interleaved, vec):
        if rot and not interleaved:
            return rot // 2 // vec + _ceil(dim - rot, 2 * vec)
        return _ceil(dim, 2 * vec)

    @staticmethod
    def _widest(itemsize, dim, rot, interleaved):
        for vec in (8, 4, 2):
            if vec * itemsize <= 16 and dim % vec == 0 and rot % (vec if interleaved else 2 * vec) == 0:
                return vec
        return 1

    def additions(self, role):
        """Additions behind an item of a weight's gradient: a lane's rows one after the other, the
        groups of a warp and the warps of a block, then a column of partial rows in four strands of
        32 warps, joined by seven more."""
        return self.rounds * self.heads_an_item[role] + 5 + 4 + _ceil(self.blocks, 128) + 2 + 5
