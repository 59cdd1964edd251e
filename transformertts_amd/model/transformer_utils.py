"""Host-side constants of the hot path (reference model/transformer_utils.py:5-21).

The sinusoid table is an init-time constant: computed once in float64 numpy exactly as the
reference does (exponent 2*(i//2)/float32(model_dim), sin on even columns, cos on odd columns) and
cast to float32; the kernels only read it.  The padding masks of transformer_utils.py:24-32 are
device kernels (ttsmi_token_pad_mask / ttsmi_length_pad_mask)."""
import numpy as np


def get_angles(pos, i, model_dim):
    return pos * (1.0 / np.power(10000, (2 * (i // 2)) / np.float32(model_dim)))


def positional_encoding(position: int, model_dim: int) -> np.ndarray:
    """[position, model_dim] float32 (the reference adds a leading broadcast axis)."""
    ang = get_angles(np.arange(position)[:, None], np.arange(model_dim)[None, :], model_dim)
    ang[:, 0::2] = np.sin(ang[:, 0::2])
    ang[:, 1::2] = np.cos(ang[:, 1::2])
    return ang.astype(np.float32)


def rotary_frequencies(dim: int, base: float = 10000.0, scaling: str = 'none', factor: float = 1.0,
                       original_length: int = 4096, slow_turns: float = 1.0, fast_turns: float = 32.0) -> np.ndarray:
    """[dim / 2] float64: radians per position of the pairs that ops.rotary turns, w_i = base^(-2 i / dim).  For contexts
    `factor` times longer than the `original_length` a model was trained on:
      'linear'  every frequency divided by the factor (positions squeezed into the trained range);
      'base'    the base raised to base * factor^(dim / (dim - 2)): the slowest pair is divided by the factor, the fastest kept;
      'bands'   pairs that make at least `fast_turns` turns over the original length kept, those with at most `slow_turns`
                divided by the factor, a linear ramp over the turns in between."""
    if dim <= 0 or dim % 2:
        raise ValueError(f'rotary_frequencies: {dim} elements (an even number)')
    if scaling not in ('none', 'linear', 'base', 'bands'):
        raise ValueError(f'rotary_frequencies: unknown scaling {scaling!r}')
    if not factor > 0 or not base > 0:
        raise ValueError('rotary_frequencies: base and factor must be positive')
    if scaling == 'base' and dim > 2:
        base = base * factor ** (dim / (dim - 2))
    freqs = float(base) ** (-np.arange(0, dim, 2, dtype=np.float64) / dim)
    if scaling == 'linear':
        freqs = freqs / factor
    if scaling == 'bands':
        if not fast_turns > slow_turns:
            raise ValueError('rotary_frequencies: fast_turns must exceed slow_turns')
        kept = np.clip((original_length * freqs / (2 * np.pi) - slow_turns) / (fast_turns - slow_turns), 0.0, 1.0)
        freqs = freqs * kept + freqs / factor * (1.0 - kept)
    return freqs
