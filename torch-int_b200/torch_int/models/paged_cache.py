"""Paged int8 key/value cache for the Int8 OPT decoder: sequences of unequal lengths in one batch.

The static cache (kv_cache.py) is one rectangular tensor per layer: every sequence has the same length and takes
its full capacity from the start.  Here, per layer, keys and values are pools of pages [num_pages, Hl, page_size, D];
a sequence holds a list of pages, the same ones in every layer, that grows a page at a time, and a step may bring
any number of new tokens for any of the sequences (a prompt, a chunk of one, single tokens).  The lists and the
lengths live on the host; a ``PagedStep`` carries what a step's kernels read to the device in one copy.
"""
from dataclasses import dataclass

import torch


@dataclass
class PagedStep:
    """A ragged batch of new tokens on the device: sequence b's are query_starts[b] .. query_starts[b + 1]."""
    query_starts: torch.Tensor   # int32 [B + 1]
    kv_lens: torch.Tensor        # int32 [B], keys once the new tokens are appended
    block_table: torch.Tensor    # int32 [B, width]
    positions: torch.Tensor      # int32 [N], position of each new token
    last: torch.Tensor           # int32 [B], index of each sequence's last new token
    max_query_len: int
    max_kv_len: int              # bound of kv_lens; raise it to the last length before capturing a step
    longest: int                 # of kv_lens

    def advance(self):
        """The next step of single tokens, on the current stream: every sequence one position further, into pages that
        are reserved (PagedInt8KVCache.reserve before the step that is advanced; a sequence without a page for its
        position is skipped, and the status word says so).  The cache's own lengths do not follow: see
        PagedInt8KVCache.fill."""
        if self.max_query_len != 1:
            raise ValueError(f"only a step of single tokens can be advanced, this one brings up to {self.max_query_len}")
        self.longest += 1
        self.max_kv_len = max(self.max_kv_len, self.longest)
        self.kv_lens.add_(1)
        self.positions.add_(1)


class PagedInt8KVCache:
    def __init__(self, num_layers, num_pages, local_heads, head_dim, device, page_size=16):
        if page_size not in (16, 32, 64, 128, 256):
            raise ValueError(f"page_size must be 16, 32, 64, 128 or 256, got {page_size}")
        if num_pages <= 0:
            raise ValueError(f"num_pages must be positive, got {num_pages}")
        self.page_size = page_size
        self.num_pages = num_pages
        self.device = torch.device(device)
        shape = (num_pages, local_heads, page_size, head_dim)
        self.k_pages = [torch.zeros(shape, dtype=torch.int8, device=device) for _ in range(num_layers)]
        self.v_pages = [torch.zeros(shape, dtype=torch.int8, device=device) for _ in range(num_layers)]
        self._free = list(range(num_pages - 1, -1, -1))
        self._pages = {}    # sequence -> its pages in order
        self._lengths = {}  # sequence -> positions filled once the last step that names it has run
        self._next = 0

    @property
    def free_pages(self):
        return len(self._free)

    def length(self, seq):
        return self._lengths[seq]

    def open(self):
        """A new, empty sequence; returns its handle."""
        seq, self._next = self._next, self._next + 1
        self._pages[seq], self._lengths[seq] = [], 0
        return seq

    def close(self, seq):
        """Gives the pages of `seq` back.  They may be handed out again at once: steps run in stream order."""
        self._free.extend(reversed(self._pages.pop(seq)))
        del self._lengths[seq]

    def reserve(self, lengths):
        """Pages for sequences to grow to `lengths` ({sequence: positions}); raises, and changes nothing, if there
        are not enough."""
        need = {s: -(-n // self.page_size) - len(self._pages[s]) for s, n in lengths.items()}
        total = sum(n for n in need.values() if n > 0)
        if total > len(self._free):
            raise RuntimeError(f"the paged cache has {len(self._free)} free pages of {self.page_size} positions, "
                               f"{total} are needed")
        for s, n in need.items():
            for _ in range(n):
                self._pages[s].append(self._free.pop())

    def step(self, seqs, new_tokens):
        """The step that appends new_tokens[i] tokens to seqs[i] (a sequence at most once).  Reserves their pages and
        counts them as filled."""
        if len(seqs) != len(new_tokens) or not seqs:
            raise ValueError("step needs one number of new tokens per sequence, and a sequence")
        if len(set(seqs)) != len(seqs):
            raise ValueError("a sequence may appear once in a step")
        if min(new_tokens) < 1:
            raise ValueError("every sequence of a step brings at least one token")
        lens = [self._lengths[s] + t for s, t in zip(seqs, new_tokens)]
        self.reserve(dict(zip(seqs, lens)))
        width = max(len(self._pages[s]) for s in seqs)
        starts, positions, table = [0], [], []
        for s, t, n in zip(seqs, new_tokens, lens):
            starts.append(starts[-1] + t)
            positions.extend(range(n - t, n))
            table.extend(self._pages[s] + [-1] * (width - len(self._pages[s])))
            self._lengths[s] = n
        b, n = len(seqs), starts[-1]
        flat = torch.tensor(starts + lens + [x - 1 for x in starts[1:]] + positions + table, dtype=torch.int32)
        if self.device.type == "cuda":
            flat = flat.pin_memory().to(self.device, non_blocking=True)
        cuts = [b + 1, b, b, n, b * width]
        starts_t, lens_t, last, pos, tab = torch.split(flat, cuts)
        return PagedStep(starts_t, lens_t, tab.view(b, width), pos, last, max(new_tokens), max(lens), max(lens))

    def fill(self, seq, length):
        """Counts the positions of `seq` up to `length` as filled: by steps that were advanced on the device."""
        if not self._lengths[seq] <= length <= len(self._pages[seq]) * self.page_size:
            raise ValueError(f"sequence {seq} has {self._lengths[seq]} positions and {len(self._pages[seq])} pages of "
                             f"{self.page_size}, cannot be filled to {length}")
        self._lengths[seq] = length

    def rewind(self, seq, length):
        """Forgets the positions of `seq` from `length` on (rejected drafts); their pages stay with it."""
        if not 0 <= length <= self._lengths[seq]:
            raise ValueError(f"sequence {seq} has {self._lengths[seq]} positions, cannot be rewound to {length}")
        self._lengths[seq] = length
