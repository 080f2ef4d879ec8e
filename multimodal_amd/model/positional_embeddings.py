"""Rotary embedding tables (megatron/model/positional_embeddings.py:38-63).  The table is built with the reference's
own arithmetic - including its quirk that, once the engine has cast the module, `inv_freq` and the positions are in
the module dtype (bf16 positions above 256 are rounded) - and handed to the HIP kernel as an input."""
import torch

from .. import _streams


class RotaryEmbedding(torch.nn.Module):
    def __init__(self, dim, base=10000, precision=torch.half):
        super().__init__()
        inv_freq = 1.0 / (base ** (torch.arange(0, dim, 2).float() / dim))
        self.register_buffer("inv_freq", inv_freq)
        self.dim = dim
        self.seq_len_cached = None
        self.cos_cached = None
        self.sin_cached = None
        self.precision = precision
        self._stamp = None  # event behind the kernels that filled the cache (multimodal_amd/_streams.py)
        self._kept = {}     # tables of generation: key -> (inv_freq, its version, cos, sin, event)
        self._replaced = []  # those of frequencies the module no longer holds

    def __getstate__(self):
        """A copy (copy.deepcopy, pickle) makes its own tables: the events behind these can be neither copied nor saved."""
        return {**self.__dict__, "seq_len_cached": None, "cos_cached": None, "sin_cached": None, "_stamp": None, "_kept": {}, "_replaced": []}

    def _build(self, x, seq_len):
        t = torch.arange(seq_len, device=x.device).type_as(self.inv_freq)
        freqs = torch.einsum("i,j->ij", t, self.inv_freq.to(x.device))
        emb = torch.cat((freqs, freqs), dim=-1).to(x.device)
        if self.precision == torch.bfloat16:
            emb = emb.float()
        cos, sin = emb.cos()[:, None, None, :], emb.sin()[:, None, None, :]
        if self.precision == torch.bfloat16:
            cos, sin = cos.bfloat16(), sin.bfloat16()
        return cos, sin

    def forward(self, x, seq_dim=1, seq_len=None):
        """Returns (cos, sin) as [seq_len, 1, 1, dim] like the reference."""
        if seq_len is None:
            seq_len = x.shape[seq_dim]
        if seq_len != self.seq_len_cached or self.cos_cached is None or self.cos_cached.device != x.device:
            self.seq_len_cached = seq_len
            self.cos_cached, self.sin_cached = self._build(x, seq_len)
            self._stamp = _streams.stamp(x.device) if x.is_cuda else None
        elif self._stamp is not None:
            _streams.wait(self._stamp, x.device)
        return self.cos_cached, self.sin_cached

    def kept_tables(self, x, positions):
        """[positions, dim] contiguous tables in x.dtype that stay where they are: generation's lengths change from call to call, and
        a captured step (of training with the tables of `forward`, of generation with these) goes on reading the ones it was
        captured with.  One pair for each power of two; new ones once the module holds other frequencies (another tensor, or a
        version counted on: whatever a load or a cast does), the old ones kept for the steps captured with them."""
        length = 1 << (positions - 1).bit_length() if positions > 1 else 1
        inv = self.inv_freq
        key = (length, x.dtype, x.device, self.precision)
        version = None if inv.is_inference() else inv._version  # None: changes are not counted, so nothing is kept
        entry = self._kept.get(key)
        if entry is not None and entry[0] is inv and entry[1] == version and version is not None:
            if entry[4] is not None:
                _streams.wait(entry[4], x.device)
            return entry[2][:positions], entry[3][:positions]
        cos, sin = (t.reshape(length, self.dim).to(x.dtype).contiguous() for t in self._build(x, length))
        # inside a capture nothing has been computed yet
        if version is not None and not (x.is_cuda and torch.cuda.is_current_stream_capturing()):
            if entry is not None:
                self._replaced.append(entry)
            self._kept[key] = (inv, version, cos, sin, _streams.stamp(x.device) if x.is_cuda else None)
        return cos[:positions], sin[:positions]

    def tables(self, x, seq_len):
        """[seq_len, dim] contiguous tables in x.dtype for the kernel."""
        cos, sin = self.forward(x, seq_len=seq_len)
        return cos.reshape(seq_len, self.dim).to(x.dtype).contiguous(), sin.reshape(seq_len, self.dim).to(x.dtype).contiguous()
