"""The tensors of a cache in pages (no counterpart in the reference)."""
from dataclasses import dataclass

import torch

BLOCK = 32  # tokens that lie together in a page


@dataclass
class PagedCache:
    """Keys and values of B sequences in pages of 8-bit codes.

    keys (pages, Hk, page / 32, Dr / 16, 32, 16) and values (pages, Hk, page / 32, Dr, 32),
    float8_e4m3fn, Dr the head size D rounded up to 16: blocks of 32 tokens, of which sixteen
    values of a key and 32 tokens of a value lie together.  key_scales and value_scales (pages,
    Hk) float32: a value is its code times the scale of its page and head.  table (B, M) int32:
    the pages of each sequence in order, -1 where there is none.  lengths (B) int64: the tokens of
    each sequence, to which a program adds the new ones before cache_append and cached_attention.
    More than the M pages of a sequence hold counts as what they hold: tokens appended beyond
    would take the places of its last ones, so a program ends a sequence before that.

    All are plain tensors that the program owns: it hands out pages by writing to `table`, and
    frees a sequence by setting its length to 0 and its entries to -1.
    """

    keys: torch.Tensor
    values: torch.Tensor
    key_scales: torch.Tensor
    value_scales: torch.Tensor
    table: torch.Tensor
    lengths: torch.Tensor

    @classmethod
    def empty(cls, sequences, longest, heads, size, page=64, pages=None, device=None):
        """A cache for `sequences` of up to `longest` tokens, with `heads` key heads of `size`.

        pages None: as many as all sequences together can need, handed out in order; else a pool
        of that many, and a table without entries.
        """
        if page < BLOCK or page > 256 or page % BLOCK != 0:
            raise ValueError(f"page must be 32 to 256 in steps of 32, but got {page}")
        if sequences < 0 or longest < 0 or heads < 1 or not 1 <= size <= 128:
            raise ValueError(f"bad sizes: {sequences} sequences of {longest} tokens, {heads} heads "
                             f"of {size} (1 to 128)")
        most = -(-longest // page)
        table = torch.arange(sequences * most, dtype=torch.int32, device=device)
        if pages is None:
            pages = sequences * most
        else:
            table = torch.full_like(table, -1)
        rounded = -(-size // 16) * 16
        kw = {"dtype": torch.uint8, "device": device}
        code = torch.float8_e4m3fn
        return cls(
            torch.zeros(pages, heads, page // BLOCK, rounded // 16, BLOCK, 16, **kw).view(code),
            torch.zeros(pages, heads, page // BLOCK, rounded, BLOCK, **kw).view(code),
            torch.ones(pages, heads, device=device), torch.ones(pages, heads, device=device),
            table.view(sequences, most),
            torch.zeros(sequences, dtype=torch.int64, device=device))

    @property
    def page(self):
        """Tokens of a page."""
        return self.keys.shape[2] * BLOCK

    def rows(self):
        """What the pages hold, in float32: keys and values (pages, Hk, page, Dr)."""
        pages, heads = self.keys.shape[:2]
        k = self.keys.float().transpose(3, 4).reshape(pages, heads, self.page, -1)
        v = self.values.float().transpose(3, 4).reshape(pages, heads, self.page, -1)
        return k * self.key_scales[..., None, None], v * self.value_scales[..., None, None]
