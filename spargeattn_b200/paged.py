"""A paged key/value cache: writing new tokens, attention over it, and the bookkeeping of its pages, all on the device.

The cache is plain tensors that the program owns:

  k_pages, v_pages  [pages, kv_heads, page_size, D] fp16 or bf16, page_size a power of two from 16 to 256; any strides with dense
                    16-byte aligned rows (a layer of one tensor [layers, 2, pages, ...], or token-major pages seen
                    through a transpose). The calls that move pages take one tensor `pages` [..., pages, kv_heads, page_size, D]
                    with all that a page number stands for (every layer's keys and values), each page one block of memory,
                    heads or tokens first: a program that forks or compacts keeps its cache in one tensor
  page_table        [sequences, width] int32: the pages of each sequence in order, -1 behind them
  seq_lens          [sequences] int32: tokens held
  ref_counts        [pages] int32: how many sequences hold a page, 0: free

A step: `allocate_pages` grows the sequences (seq_lens then include the new tokens) and says which it served, and each layer calls
`append_kv`, with that, and `paged_attention`. New tokens are packed, [tokens, heads, D]: sequence i has the rows cu_seqlens[i] to
cu_seqlens[i + 1], its last tokens; without cu_seqlens every sequence has one. No function synchronises or copies to the host,
and lengths, tables and cu_seqlens are read when the kernels run, so a captured step follows them from replay to replay.

Lengths grow by `allocate_pages` and go back to 0 by `free_sequences`. A program that lowers one itself (drafted tokens that were
rejected) also sets the entries of the pages behind it to -1 and takes one off their counts: `allocate_pages` writes over
what stands there, and a page whose entry is gone keeps its count. It does not go back into a page that a fork shares: the next
token would be written for both.

Arguments that do not fit are ValueError, CPU tensors RuntimeError. What only the device can see (a page number outside the
pool, a length outside the table) is skipped without touching other memory and reported through `ops.check_device_status()`; the
first report stays until `ops.device_status_word(device).zero_()`.
Nothing here has a gradient. The first call on a device should precede graph capture: it sets up the word that reports go to.
"""
import torch

from . import ops
from ._cabi import _binding

# the tracing compiler leaves these frames alone, which costs a call nothing
_skip_frame = torch.compiler.disable(recursive=False)


def _status(t):
    """The device's status word exists before a kernel may want to write to it."""
    if isinstance(t, torch.Tensor) and t.is_cuda and t.device.index not in ops._status_words:
        ops.device_status_word(t.device)


@_skip_frame
def append_kv(k, v, k_pages, v_pages, page_table, seq_lens, cu_seqlens=None, q=None, frequencies=None, interleaved=False,
              magnitude=1.0, served=None):
    """Writes the new tokens' k and v [tokens, kv_heads, D] to their pages. seq_lens include them.

    With `frequencies` (see `apply_rotary`) k is turned by its position in the sequence on the way, and q [tokens, heads, D], if
    given, is turned too and returned (rows of no sequence: zeros): one pass over the layer's projections. Else returns
    None. A token whose position has no page is left out and reported.

    `served` [sequences] bool, as `allocate_pages` returned it, leaves out the tokens of sequences that it did not serve (their q
    becomes zeros, and what attention makes of that means nothing). Where the pool or a row of the table may run out it is needed:
    such a sequence kept its length, so its tokens would fall on its last positions, over keys that it holds, and that
    its forks may share. Sequences that share the page they write to otherwise (a served sequence never does, after
    `fork_sequences` and `allocate_pages`) are the caller's mistake."""
    _status(k)
    return _binding.append_kv(k, v, k_pages, v_pages, page_table, seq_lens, cu_seqlens, q, frequencies, interleaved, magnitude, served)


@_skip_frame
def paged_attention(q, k_pages, v_pages, page_table, seq_lens, cu_seqlens=None, max_chunk=None, is_causal=True, scale=None, out=None,
                    return_lse=False):
    """Attention of the new tokens' q [tokens, heads, D] over all that their sequences hold: out, or (out, lse [tokens, heads] fp32).

    Query head h reads key head h // (heads // kv_heads). Token j of a sequence's n new ones sees the keys up to its own position
    seq_len - n + j (`is_causal=False`: all of the sequence's). A row that sees no key gives zeros and an lse of -inf. D is 64
    or 128, scale defaults to D ** -0.5. `max_chunk`, an upper bound of the new tokens of one sequence, chooses the kernel
    (without it: all tokens, or 1 without cu_seqlens); results hold whatever it says. Rows of no sequence are zeros, or left as
    they were in a given `out`; their lse is -inf. What pages hold behind the length never reaches a result; an infinity or NaN
    in V at a position that a row does not see but a later row of its chunk does may (0 * inf), as it does in a masked product."""
    _status(q)
    return _binding.paged_attention(q, k_pages, v_pages, page_table, seq_lens, cu_seqlens, max_chunk, is_causal, scale, out, return_lse)


@_skip_frame
def allocate_pages(page_table, seq_lens, ref_counts, new_tokens, page_size):
    """Room for new_tokens [sequences] int32 more tokens each, in place: seq_lens grow, and new pages (lowest free first, for one
    sequence after the other) enter the table with a count of 1. Returns served [sequences] bool: a sequence that its row or
    the pool has no room for keeps its length and gets nothing; behind the first one that the pool cannot serve only those that
    need no page are served."""
    return _binding.allocate_pages(page_table, seq_lens, ref_counts, new_tokens, page_size)


@_skip_frame
def free_sequences(page_table, seq_lens, ref_counts, sequences, page_size=None):
    """Empties these sequences' rows (int32 numbers; -1 is skipped, a number twice is freed once): their pages lose a count, their
    lengths become 0. `page_size` is not needed and accepted for symmetry with `allocate_pages`."""
    _status(page_table)
    return _binding.free_sequences(page_table, seq_lens, ref_counts, sequences)


@_skip_frame
def fork_sequences(pages, page_table, seq_lens, ref_counts, src, dst):
    """Sequence dst[i] becomes a copy of sequence src[i], for all i at once (a permutation of beams is fine). Full pages are
    shared; a last page that is not full is copied to a fresh one, in every layer that `pages` [..., pages, kv_heads, page_size, D]
    holds, so that both may go on writing. What the destinations held is released afterwards. Returns served [len(src)] bool: False
    where no page was left (the destination stays as it was), where the pair is skipped (-1), or where a later pair that is not
    skipped has the same destination."""
    _status(pages)
    return _binding.fork_sequences(pages, page_table, seq_lens, ref_counts, src, dst)


@_skip_frame
def compact_pages(pages, page_table, ref_counts):
    """Moves the pages in use (a count above 0) to the front of the pool, in every layer that `pages` holds, and rewrites table and
    counts in place. Returns their number, int32 [1] on the device: pages from there on are free. A page that the program holds by
    a count of its own, without an entry of the table, moves like the others."""
    return _binding.compact_pages(pages, page_table, ref_counts)


@_skip_frame
def copy_pages(pages, src, dst):
    """Page dst[i] becomes a copy of page src[i] in every layer that `pages` holds; pairs with -1 are skipped. A pair whose
    destination is the destination or source of another one that is not skipped has no defined order: it is not copied, and
    reported."""
    _status(pages)
    return _binding.copy_pages(pages, src, dst)
