"""The cache operators where no GPU is needed: what they refuse, their frequencies, and how attention cuts its work."""
import ctypes
import math
import os
import shutil
import subprocess

import pytest
import torch

import spargeattn_b200 as S
from spargeattn_b200 import _cabi

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "spargeattn_b200", "csrc")
BF = torch.bfloat16


def _cache(S_=2, W=4, P=8, H=2, ps=16, D=64, dtype=BF):
    return dict(k_pages=torch.zeros(P, H, ps, D, dtype=dtype), v_pages=torch.zeros(P, H, ps, D, dtype=dtype),
                page_table=torch.zeros(S_, W, dtype=torch.int32), seq_lens=torch.ones(S_, dtype=torch.int32))


def _freq(n):
    return torch.ones(n, dtype=torch.float64)


@pytest.mark.parametrize("change,text", [
    (dict(tensor_layout="DNH"), "tensor_layout"), (dict(positions=torch.zeros(5, dtype=torch.float32)), "int32 or int64"),
    (dict(positions=torch.zeros(4, dtype=torch.int32)), "tokens"), (dict(frequencies=_freq(40)), "frequencies"),
    (dict(frequencies=torch.ones(8)), "float64"), (dict(sections=[3, 4], positions=torch.zeros(2, 5, dtype=torch.int32)), "add up"),
    (dict(sections=[4, 4]), "positions"), (dict(sections=[4, -4, 8], positions=torch.zeros(3, 5, dtype=torch.int32)), "add up"),
    (dict(sections=[2, 2, 2, 1, 1], positions=torch.zeros(5, 5, dtype=torch.int32)), "1 to 4"),
    (dict(k=torch.zeros(1, 3, 6, 64, dtype=BF)), "but for the heads"), (dict(k=torch.zeros(1, 3, 5, 64)), "type"),
    (dict(q=torch.zeros(5, 64, dtype=BF)), "dimensions"), (dict(q=torch.zeros(1, 2, 5, 64, dtype=torch.float64)), "float16"),
    (dict(magnitude=math.inf), "finite")])
def test_rotary_refuses(change, text):
    a = dict(q=torch.zeros(1, 2, 5, 64, dtype=BF), k=torch.zeros(1, 3, 5, 64, dtype=BF), positions=torch.zeros(5, dtype=torch.int32),
             frequencies=_freq(8)) | change
    with pytest.raises(ValueError, match=text):
        S.apply_rotary(**a)


def test_cpu_tensors_are_refused():
    q = torch.zeros(2, 4, 64, dtype=BF)
    table, lens, refs = torch.zeros(2, 4, dtype=torch.int32), torch.ones(2, dtype=torch.int32), torch.zeros(8, dtype=torch.int32)
    one = torch.zeros(1, dtype=torch.int32)
    pool = torch.zeros(2, 8, 2, 16, 64, dtype=BF)
    for call in (lambda: S.apply_rotary(q, None, lens, _freq(8), tensor_layout="NHD"), lambda: S.paged_attention(q, **_cache()),
                 lambda: S.append_kv(q[:, :2], q[:, :2], **_cache()), lambda: S.allocate_pages(table, lens, refs, lens, 16),
                 lambda: S.free_sequences(table, lens, refs, one), lambda: S.fork_sequences(pool, table, lens, refs, one, one),
                 lambda: S.compact_pages(pool, table, refs), lambda: S.copy_pages(pool, one, one)):
        with pytest.raises(RuntimeError, match="CUDA tensors only"):
            call()


@pytest.mark.parametrize("change,text", [
    (dict(q=torch.zeros(2, 3, 64, dtype=BF)), "multiple"), (dict(q=torch.zeros(2, 4, 128, dtype=BF)), "head_dim"),
    (dict(q=torch.zeros(2, 4, 64, dtype=torch.float16)), "type"), (dict(q=torch.zeros(3, 4, 64, dtype=BF)), "one token"),
    (dict(k_pages=torch.zeros(8, 2, 24, 64, dtype=BF), v_pages=torch.zeros(8, 2, 24, 64, dtype=BF)), "page_size"),
    (dict(k_pages=torch.zeros(9, 2, 16, 64, dtype=BF)), "same shape"), (dict(seq_lens=torch.ones(3, dtype=torch.int32)), "seq_lens"),
    (dict(seq_lens=torch.ones(2, dtype=torch.int64)), "int32"), (dict(page_table=torch.zeros(2, 4, dtype=torch.int64)), "int32"),
    (dict(cu_seqlens=torch.zeros(2, dtype=torch.int32)), "cu_seqlens"), (dict(max_chunk=-1), "max_chunk"), (dict(scale=math.nan), "scale"),
    (dict(out=torch.zeros(2, 4, 64)), "out"), (dict(out=torch.zeros(2, 1, 64, dtype=BF).expand(2, 4, 64)), "apart"),
    (dict(k_pages=torch.zeros(1, 2, 16, 64, dtype=BF).expand(8, 2, 16, 64)), "apart"), (dict(q=torch.zeros(2, 4, 65, dtype=BF)[..., 1:]), "aligned"),
    (dict(k_pages=torch.zeros(8, 2, 16, 96, dtype=BF), v_pages=torch.zeros(8, 2, 16, 96, dtype=BF)), "headdim"),
    (dict(k_pages=torch.zeros(0, 2, 16, 64, dtype=BF), v_pages=torch.zeros(0, 2, 16, 64, dtype=BF)), "no pages")])
def test_attention_refuses(change, text):
    with pytest.raises(ValueError, match=text):
        S.paged_attention(**(dict(q=torch.zeros(2, 4, 64, dtype=BF)) | _cache() | change))


@pytest.mark.parametrize("change,text", [
    (dict(v=torch.zeros(2, 3, 64, dtype=BF)), "one shape"), (dict(k=torch.zeros(2, 1, 64, dtype=BF), v=torch.zeros(2, 1, 64, dtype=BF)), "heads"),
    (dict(q=torch.zeros(2, 4, 64, dtype=BF)), "frequencies"), (dict(q=torch.zeros(3, 4, 64, dtype=BF), frequencies=_freq(8)), "tokens"),
    (dict(frequencies=_freq(33)), "frequencies"), (dict(k=torch.zeros(3, 2, 64, dtype=BF), v=torch.zeros(3, 2, 64, dtype=BF)), "one token")])
def test_append_refuses(change, text):
    with pytest.raises(ValueError, match=text):
        S.append_kv(**(dict(k=torch.zeros(2, 2, 64, dtype=BF), v=torch.zeros(2, 2, 64, dtype=BF)) | _cache() | change))


def test_bookkeeping_refuses():
    table, lens, refs = torch.zeros(2, 4, dtype=torch.int32), torch.ones(2, dtype=torch.int32), torch.zeros(8, dtype=torch.int32)
    one, pool = torch.zeros(1, dtype=torch.int32), torch.zeros(2, 8, 2, 16, 64, dtype=BF)
    for call, text in ((lambda: S.allocate_pages(table, lens, refs, one, 16), "new_tokens"), (lambda: S.allocate_pages(table, lens, refs, lens, 20), "page_size"),
                       (lambda: S.allocate_pages(table.long(), lens, refs, lens, 16), "int32"), (lambda: S.allocate_pages(table, one, refs, lens, 16), "seq_lens"),
                       (lambda: S.allocate_pages(table[:1].expand(2, 4), lens, refs, lens, 16), "overlap"),
                       (lambda: S.free_sequences(table, lens, refs.long(), one), "ref_counts"), (lambda: S.free_sequences(table, lens, refs, one.long()), "sequences"),
                       (lambda: S.fork_sequences(pool[:, :7], table, lens, refs, one, one), "each of the 7"), (lambda: S.fork_sequences(pool, table, lens, refs, one, lens), "dst"),
                       (lambda: S.compact_pages(pool.transpose(2, 3), table, refs), "one block"), (lambda: S.copy_pages(pool, one, lens), "dst"),
                       (lambda: S.copy_pages(pool, torch.zeros(65537, dtype=torch.int32), torch.zeros(65537, dtype=torch.int32)), "at most 65536"),
                       (lambda: S.fork_sequences(pool, table, lens, refs, torch.zeros(65537, dtype=torch.int32), torch.zeros(65537, dtype=torch.int32)), "at most"),
                       (lambda: S.copy_pages(pool[0, 0], one, one), "pages"), (lambda: S.copy_pages(pool[:, :, :, ::2], one, one), "one block")):
        with pytest.raises(ValueError, match=text):
            call()
    with pytest.raises(TypeError):
        S.copy_pages(None, one, one)


def test_c_entries_check_their_arguments():
    L, one = _cabi.lib, ctypes.c_void_p(16)
    assert L.sparge_rotary(None, None) == L.sparge_append_kv(None, None) == L.sparge_paged_attention(None, None) == _cabi.ERR_NULL
    zeros = ctypes.create_string_buffer(1024)       # sizes of zero: refused before any pointer is looked at
    for f in (L.sparge_rotary, L.sparge_append_kv, L.sparge_paged_attention):
        assert f(zeros, None) == _cabi.ERR_INVALID_ARG
    assert L.sparge_paged_attention_workspace_bytes(6, 4, 64, 1) == 0 and L.sparge_paged_attention_workspace_bytes(8, 4, 64, 1) > 0
    assert L.sparge_allocate_pages(one, one, one, None, one, one, 2, 4, 4, 8, 16, None) == _cabi.ERR_NULL
    assert L.sparge_allocate_pages(one, one, one, one, one, one, 2, -1, 4, 8, 16, None) == _cabi.ERR_INVALID_ARG
    assert L.sparge_free_sequences(one, one, one, None, 1, 2, 4, 4, 8, None, None) == _cabi.ERR_NULL
    assert L.sparge_copy_pages(one, 1, 0, 64, 24, one, one, 1, 8, None, None) == _cabi.ERR_INVALID_ARG      # pages of 24 bytes
    assert L.sparge_copy_pages(one, 1, 0, 64, 32, one, one, 65537, 8, None, None) == _cabi.ERR_TOO_LARGE
    assert L.sparge_copy_pages(None, 1, 0, 64, 32, one, one, 1, 8, None, None) == _cabi.ERR_NULL
    assert L.sparge_compact_pages(one, 1, 0, 32, 32, one, one, None, one, 1, 4, 4, 8, None) == _cabi.ERR_NULL
    assert L.sparge_fork_sequences(one, 1, 0, 32, 32, one, one, one, one, None, one, one, 1, 2, 4, 4, 8, 16, None, None) == _cabi.ERR_NULL


def test_frequencies():
    f, m = S.rotary_frequencies(64, 10000.0, device="cpu")
    i = torch.arange(32, dtype=torch.float64)
    assert f.dtype == torch.float64 and m == 1.0
    assert torch.allclose(f, 1 / 10000.0 ** (i / 32), rtol=1e-14)
    assert torch.allclose(S.rotary_frequencies(64, scaling="linear", factor=4, device="cpu")[0], f / 4, rtol=1e-14)
    ntk = S.rotary_frequencies(64, scaling="ntk", factor=8, device="cpu")[0]
    assert ntk[0] == 1.0 and math.isclose(ntk[-1], f[-1] / 8, rel_tol=1e-12)
    turns = 8192 * f / (2 * math.pi)
    l3 = S.rotary_frequencies(64, scaling="llama3", factor=8, original_length=8192, device="cpu")[0]
    assert torch.equal(l3[turns >= 4], f[turns >= 4]) and torch.allclose(l3[turns <= 1], f[turns <= 1] / 8, rtol=1e-14)
    assert (l3 <= f).all() and (l3 >= f / 8 * (1 - 1e-14)).all()
    y, m = S.rotary_frequencies(64, scaling="yarn", factor=8, original_length=8192, device="cpu")
    assert torch.equal(y[turns >= 64], f[turns >= 64]) and torch.allclose(y[turns <= 0.5], f[turns <= 0.5] / 8, rtol=1e-14)
    assert math.isclose(m, 0.1 * math.log(8) + 1)
    for bad in (dict(dim=5), dict(dim=0), dict(dim=8, scaling="x"), dict(dim=8, scaling="yarn"), dict(dim=8, factor=0.5),
                dict(dim=8, scaling="llama3", original_length=100, low=4, high=4), dict(dim=2, scaling="ntk"), dict(dim=8, base=1.0)):
        with pytest.raises(ValueError):
            S.rotary_frequencies(**bad, device="cpu")


def test_shares_of_attention(tmp_path):
    """Blocks of a sequence's tiles by the closed form are those counted one by one, and shares cover the line evenly."""
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("no g++")
    src = tmp_path / "schedule.cpp"
    src.write_text('''
#include <initializer_list>
#include "paged_schedule.cuh"
using namespace sparge;
template <int ROWS>
int check() {
  for (unsigned group : {1, 2, 3, 5, 8, 12, 40, 128})
    for (bool causal : {false, true})
      for (unsigned tokens : {1, 2, 7, 16, 31, 100, 333, 1000})
        for (unsigned length : {0, 1, 5, 100, 127, 128, 129, 333, 1000, 1001, 5003}) {
          const SeqWork<ROWS> w{tokens, length, group, causal};
          long long sum = 0, all = 0;
          for (unsigned t = 0; t < w.tiles(); t++) {
            if (w.blocks_before(t) != sum || w.blocks(t) < 1) return 1;
            sum += w.blocks(t);
            // every key that a row of the tile sees lies in its blocks
            for (unsigned r = 0; r < w.tile_rows(t); r++)
              if (w.visible(t * ROWS + r) > (long long)w.blocks(t) * kBlockKeys) return 2;
            all += w.tile_rows(t);
          }
          if (w.units() != sum || all != w.all_rows()) return 3;
        }
  // a long context: no overflow
  const SeqWork<ROWS> w{1u << 20, 0x7fffff00u, 8, true};
  long long sum = 0;
  for (unsigned t = 0; t < w.tiles(); t++) sum += w.blocks(t);
  return w.units() == sum ? 0 : 4;
}
int main() {
  if (int rc = check<16>() + 10 * check<128>() + 100 * check<256>()) return rc;
  for (long long units : {1LL, 5LL, 147LL, 148LL, 1000LL, 12345678901LL})
    for (int shares : {1, 5, 148}) {
      if (shares > units) continue;
      long long at = 0, least = units, most = 0;
      for (int c = 0; c < shares; c++) {
        const long long a = share_begin(c, units, shares), b = share_begin(c + 1, units, shares);
        if (a != at || share_of(a, units, shares) != c || share_of(b - 1, units, shares) != c) return 5;
        at = b;
        least = b - a < least ? b - a : least, most = b - a > most ? b - a : most;
      }
      if (at != units || most - least > 1 || least < 1) return 6;
    }
  return 0;
}
''')
    subprocess.run([gxx, "-std=c++17", "-O2", "-I", CSRC, str(src), "-o", str(tmp_path / "schedule")], check=True)
    assert subprocess.run([str(tmp_path / "schedule")]).returncode == 0


def test_page_layouts():
    """A page that is one block is taken in either order of its heads and tokens (and then has to be on a GPU); strides of dimensions of
    one say nothing. Pages that interleave, or have gaps, are refused."""
    table, lens, one = torch.zeros(2, 4, dtype=torch.int32), torch.ones(2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)

    def calls(pool):
        refs = torch.zeros(pool.shape[-4], dtype=torch.int32)
        return (lambda: S.fork_sequences(pool, table, lens, refs, one, one), lambda: S.compact_pages(pool, table, refs),
                lambda: S.copy_pages(pool, one, one))

    flat = torch.zeros(8 * 16 * 64, dtype=BF)
    for pool in (*(torch.zeros(3, 2, 8, 16, H, 64, dtype=BF).transpose(3, 4) for H in (1, 2, 16)),
                 flat.as_strided((8, 1, 16, 64), (16 * 64, 3, 64, 1)), flat.as_strided((8, 1, 16, 64), (16 * 64, 64, 64, 1)),
                 flat.as_strided((1, 2, 16, 64), (5, 16 * 64, 64, 1)), flat.as_strided((1, 2, 16, 64), (5, 64, 128, 1))):
        for call in calls(pool):
            with pytest.raises(RuntimeError, match="CUDA tensors only"):
                call()
    for pool in (torch.zeros(2, 16, 8, 2, 64, dtype=BF).permute(0, 2, 3, 1, 4), torch.zeros(8, 2, 32, 64, dtype=BF)[:, :, ::2],
                 torch.zeros(8, 2, 17, 64, dtype=BF)[:, :, :16], torch.zeros(8, 16, 3, 64, dtype=BF).transpose(1, 2)[:, :2],
                 torch.zeros(1, 1, 1, 64, dtype=BF).expand(8, 2, 16, 64), torch.zeros(8, 2, 64, 16, dtype=BF).transpose(2, 3)):
        for call in calls(pool):
            with pytest.raises(ValueError, match="one block"):
                call()


@pytest.mark.parametrize("served,text", [(torch.ones(2, dtype=torch.int32), "bool"), (torch.ones(3, dtype=torch.bool), "sequences"),
                                         (torch.ones(2, 1, dtype=torch.bool), "bool"), (torch.ones(4, dtype=torch.bool)[::2], "bool")])
def test_append_refuses_served(served, text):
    k = torch.zeros(2, 2, 64, dtype=BF)
    with pytest.raises(ValueError, match=text):
        S.append_kv(k, k, **_cache(), served=served)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        S.append_kv(k, k, **_cache(), served=torch.ones(2, dtype=torch.bool))


def test_magnitudes_beyond_32_bits_are_refused():
    """A factor that is finite in 64 bits and infinite in the kernels' 32."""
    q, k = torch.zeros(1, 2, 5, 64, dtype=BF), torch.zeros(2, 2, 64, dtype=BF)
    for call in (lambda: S.apply_rotary(q, None, torch.zeros(5, dtype=torch.int32), _freq(8), magnitude=1e39),
                 lambda: S.append_kv(k, k, **_cache(), frequencies=_freq(8), magnitude=-1e39)):
        with pytest.raises(ValueError, match="finite"):
            call()
