"""Buckets of relative positions: what `ops.relpos_attention` needs to know about a learned position bias.

A query at position p and a key at position r share the bias table[bucket(r - p), head].  `RelPosBuckets` holds the bucket of every difference
lo .. lo + width - 1 (differences beyond the ends take the end's bucket) and, where the positions are not simply the tokens' numbers, the
positions themselves."""
import numpy as np
import torch

from .hip import OfbError, raw_stream

MAX_WIDTH = 4096
_FAR = 1 << 26                         # (four times a difference of two positions and `lo` stays a 32-bit number)


class RelPosBuckets:
    """lut: bucket of the differences lo, lo + 1, ...; num_buckets: rows of the table (default: the largest bucket + 1);
    positions: (positions of the queries, positions of the keys) as integer sequences, for sequences of exactly those lengths - default: key j
    stands at j and query i at i + q_offset.

    One plan serves any number of layers, batches, devices and streams; `to(device)` uploads it ahead of the first call (a call uploads it
    otherwise, which a captured graph cannot).  A captured graph reads the upload at every replay: keep the plan as long as the graph."""

    def __init__(self, lut, lo, num_buckets=None, positions=None):
        lut = [int(x) for x in (lut.tolist() if isinstance(lut, torch.Tensor) else lut)]
        if not lut or min(lut) < 0:
            raise OfbError('RelPosBuckets: the buckets are whole numbers from 0 on, at least one')
        lo, self.num_buckets = int(lo), int(num_buckets) if num_buckets is not None else max(lut) + 1
        if max(lut) >= self.num_buckets:
            raise OfbError(f'RelPosBuckets: bucket {max(lut)} of a table of {self.num_buckets} rows')
        if self.num_buckets > 1 << 20:
            raise OfbError('RelPosBuckets: tables of more than 2^20 rows are not supported')
        first, last = 0, len(lut) - 1                          # runs of one bucket at the ends say nothing that the clamp does not
        while first < last and lut[first + 1] == lut[0]:
            first += 1
        while last > first and lut[last - 1] == lut[-1]:
            last -= 1
        self.lut, self.lo = lut[first:last + 1], lo + first
        if len(self.lut) > MAX_WIDTH:
            raise OfbError(f'RelPosBuckets: {len(self.lut)} different differences, at most {MAX_WIDTH} are supported')
        if abs(self.lo) > _FAR:
            raise OfbError('RelPosBuckets: differences beyond 2^26 are not supported')
        self.positions = None
        if positions is not None:
            self.positions = tuple([int(x) for x in (p.tolist() if isinstance(p, torch.Tensor) else p)] for p in positions)
            if len(self.positions) != 2 or any(abs(x) > _FAR for p in self.positions for x in p):
                raise OfbError('RelPosBuckets: positions are two sequences of whole numbers within 2^26')
        self._on = {}

    def __getstate__(self):
        return dict(self.__dict__, _on={})

    def __deepcopy__(self, memo):
        return self                                            # immutable: the blocks of a model share one

    @property
    def width(self):
        return len(self.lut)

    def on(self, device):
        """(lut, bucket_start, bucket_order, positions of the queries or None, of the keys or None) as int32 tensors of `device`"""
        device = torch.device(device)
        if device.index is None and device.type == 'cuda':
            device = torch.device('cuda', torch.cuda.current_device())
        got, raw = self._on.get(device), raw_stream(device)
        if got is None:
            lut = np.asarray(self.lut)
            start = np.cumsum(np.bincount(lut, minlength=self.num_buckets))
            parts = [lut, [0], start, np.argsort(lut, kind='stable'), *(self.positions or ())]
            flat = torch.from_numpy(np.concatenate(parts).astype(np.int32)).to(device)
            sizes = [self.width, self.num_buckets + 1, self.width, *(len(p) for p in self.positions or ())]
            parts = list(flat.split(sizes))
            got = self._on[device] = (tuple(parts) if self.positions else (*parts, None, None), {raw})
            if device.type == 'cuda':
                torch.cuda.current_stream(device).synchronize()      # any stream may read the plan from here on
        tensors, streams = got
        if raw not in streams:                                 # a dropped plan's memory waits for the streams that read it
            streams.add(raw)
            tensors[0].record_stream(torch.cuda.current_stream(device))      # (one allocation holds all parts)
        return tensors

    def to(self, device):
        self.on(device)
        return self

    # ---- the usual rules -------------------------------------------------------------------------------------------------
    @classmethod
    def clipped(cls, max_distance):
        """one bucket per difference -max_distance .. max_distance, the ends for everything beyond"""
        r = int(max_distance)
        if r < 0:
            raise OfbError('clipped: max_distance is a whole number from 0 on')
        return cls(range(2 * r + 1), -r)

    @classmethod
    def log_spaced(cls, num_buckets=32, max_distance=128, bidirectional=True):
        """Distances below half of a direction's buckets have one each; the others share the distances up to max_distance in equal steps of the
        logarithm, the last bucket also taking everything beyond.  bidirectional: the lower half of the table for keys at or before the
        query, the upper half for those after it; otherwise keys after the query share bucket 0 (a causal decoder)."""
        num_buckets, max_distance = int(num_buckets), int(max_distance)
        per = num_buckets // 2 if bidirectional else num_buckets
        if per < 1 or (bidirectional and num_buckets % 2):
            raise OfbError('log_spaced: at least one bucket a direction, an even number of them for two directions')
        exact = per // 2
        if max_distance <= exact or max_distance > _FAR:
            raise OfbError(f'log_spaced: max_distance must be over {exact}, where the buckets of one distance each end')
        # first distance of bucket exact + k: the smallest n with (n / exact)^steps >= (max_distance / exact)^k, in whole numbers
        steps, by_distance, n = per - exact, list(range(exact)), exact
        for k in range(1, steps):
            while n ** steps * exact ** k < max_distance ** k * exact ** steps:
                by_distance.append(exact + k - 1)
                n += 1
                if n > MAX_WIDTH:
                    raise OfbError(f'log_spaced: distances beyond {MAX_WIDTH} are told apart, which is not supported')
        by_distance.append(per - 1)
        before = by_distance[:0:-1]                            # keys before the query, farthest first
        after = [per + c for c in by_distance[1:]] if bidirectional else [0]
        if bidirectional and len(by_distance) == 1:
            before, after = [by_distance[0]], [per + by_distance[0]]
        return cls(before + [by_distance[0]] + after, -len(before), num_buckets)

    @classmethod
    def grid(cls, height, width, cls_token=True):
        """The patches of a height x width grid, row by row: one bucket per difference (dy, dx), at row
        (dy + height - 1) (2 width - 1) + dx + width - 1 of the table; with a class token in front three more: class token to patch, patch to class token,
        class token to itself."""
        h, w = int(height), int(width)
        if h < 1 or w < 1:
            raise OfbError('grid: height and width are at least 1')
        m = (h - 1) * (2 * w - 1) + w - 1                      # y (2 w - 1) + x: its differences -m .. m tell the pairs (dy, dx) apart
        code = [y * (2 * w - 1) + x for y in range(h) for x in range(w)]
        near, n = list(range(2 * m + 1)), 2 * m + 1
        if not cls_token:
            return cls(near, -m, n, (code, code))
        far = 3 * m + 2                                        # the class token as a key; as a query m + 1 lower, a difference no patches have
        return cls([n] + near + [n + 2, n + 1], -m - 1, n + 3, ([far - m - 1] + code, [far] + code))
