//! Rows in groups: products, joins and gradients over rows that an index sorts into groups whose sizes stay on the
//! device.  An addition of the C library; the reference has no counterpart.
use std::ffi::c_void;
use std::ptr;

use tenferro_device::{Error, Result};
use tenferro_hip_sys as sys;

use crate::{check, HipBuffer, HipView, HipViewMut, Stream};

/// A bfloat16 element by its bits: the upper half of an f32's.
#[repr(transparent)]
#[derive(Clone, Copy, Debug, Default, PartialEq, Eq)]
pub struct Bf16(pub u16);

/// An IEEE binary16 element by its bits.
#[repr(transparent)]
#[derive(Clone, Copy, Debug, Default, PartialEq, Eq)]
pub struct F16(pub u16);

/// The element types of operations on rows in groups.  `Sum`: the type of their sums, which weights and scales are of.
pub trait RowScalar: Copy {
    type Sum: Copy;
    const TAG: i32;
}
impl RowScalar for Bf16 {
    type Sum = f32;
    const TAG: i32 = sys::TFH_BF16;
}
impl RowScalar for F16 {
    type Sum = f32;
    const TAG: i32 = sys::TFH_F16;
}
impl RowScalar for f32 {
    type Sum = f32;
    const TAG: i32 = sys::TFH_F32;
}
impl RowScalar for f64 {
    type Sum = f64;
    const TAG: i32 = sys::TFH_F64;
}

/// The integers that rows are grouped by.
pub trait RowIndex: Copy {
    const BITS: i32;
}
impl RowIndex for i32 {
    const BITS: i32 = 32;
}
impl RowIndex for i64 {
    const BITS: i32 = 64;
}

/// Rows listed group by group: group g is places `offsets[g]..offsets[g + 1]`, place p holds row `order[p]`, row i
/// stands at `positions[i]` (-1: in no group).
pub struct RowGroups {
    offsets: HipBuffer<i32>,
    order: HipBuffer<i32>,
    positions: HipBuffer<i32>,
    n_rows: usize,
    n_groups: usize,
    fan: usize,
    // read by kernels of the grouping call: lives as long as the groups
    _workspace: Option<HipBuffer<u8>>,
}

/// The low-rank factors of `RowGroups::adapter_gemm`: `a` [n_groups, K, R], `b` [n_groups, R, N], `scales` [n_groups].
pub struct AdapterFactors<'a, T: RowScalar> {
    pub a: &'a HipView<'a, T>,
    pub b: &'a HipView<'a, T>,
    pub scales: Option<&'a HipView<'a, T::Sum>>,
}

fn optional<T: Copy>(v: Option<&HipView<'_, T>>) -> Option<sys::tfh_view> {
    v.map(|v| v.raw())
}
fn optional_mut<T: Copy>(v: Option<&mut HipViewMut<'_, T>>) -> Option<sys::tfh_view> {
    v.map(|v| v.raw())
}
fn address(v: &Option<sys::tfh_view>) -> *const sys::tfh_view {
    v.as_ref().map_or(ptr::null(), |v| v as *const _)
}

impl RowGroups {
    /// Stable grouping by `ids` ([n_rows] or [tokens, fan]); an index outside `0..n_groups` puts its row into no group.
    pub fn from_ids<I: RowIndex>(ids: &HipView<I>, n_groups: usize, device_id: usize, stream: &Stream) -> Result<Self> {
        let n_rows: usize = ids.dims().iter().product();
        if n_groups > i32::MAX as usize {
            return Err(Error::InvalidArgument(format!("{n_groups} groups are out of range")));
        }
        let fan = if ids.dims().len() == 2 { ids.dims()[1].max(1) } else { 1 };
        let need = unsafe { sys::tfh_group_rows_workspace(n_rows as i64, n_groups as i32) };
        let workspace = if need > 0 { Some(HipBuffer::<u8>::new(need, device_id)?) } else { None };
        let groups = RowGroups {
            offsets: HipBuffer::new(n_groups + 1, device_id)?,
            order: HipBuffer::new(n_rows.max(1), device_id)?,
            positions: HipBuffer::new(n_rows.max(1), device_id)?,
            n_rows,
            n_groups,
            fan,
            _workspace: workspace,
        };
        let scratch = groups._workspace.as_ref().map_or(ptr::null_mut(), |w| w.as_device_ptr() as *mut c_void);
        let raw = ids.raw();
        check(unsafe {
            sys::tfh_group_rows(
                I::BITS,
                &raw,
                n_groups as i32,
                groups.offsets.as_device_ptr(),
                groups.order.as_device_ptr(),
                groups.positions.as_device_ptr(),
                scratch,
                need,
                stream.raw(),
            )
        })?;
        Ok(groups)
    }

    fn raw(&self) -> sys::tfh_row_groups {
        sys::tfh_row_groups {
            offsets: self.offsets.as_device_ptr(),
            order: self.order.as_device_ptr(),
            positions: self.positions.as_device_ptr(),
            n_rows: self.n_rows as i64,
            n_groups: self.n_groups as i32,
            fan: self.fan as i32,
        }
    }

    /// `c[p] = alpha * a[src(p)] . b[g(p)] + beta * c[p]`; `flags` of `TFH_ROWS_*`.
    pub fn gemm<T: RowScalar>(&self, flags: i32, alpha: f64, a: &HipView<T>, b: &HipView<T>, beta: f64, c: &mut HipViewMut<T>, stream: &Stream) -> Result<()> {
        let (g, a, b, c) = (self.raw(), a.raw(), b.raw(), c.raw());
        check(unsafe { sys::tfh_ragged_gemm(T::TAG, &g, flags, alpha, &a, &b, beta, &c, stream.raw()) })
    }

    /// `db[g] = alpha * sum over p in g of a[src(p)]^T dc[p] + beta * db[g]`.
    pub fn gemm_grad<T: RowScalar>(&self, flags: i32, alpha: f64, a: &HipView<T>, dc: &HipView<T>, beta: f64, db: &mut HipViewMut<T>, stream: &Stream) -> Result<()> {
        let (g, a, dc, db) = (self.raw(), a.raw(), dc.raw(), db.raw());
        check(unsafe { sys::tfh_ragged_gemm_grad(T::TAG, &g, flags, alpha, &a, &dc, beta, &db, stream.raw()) })
    }

    /// `da[s] = alpha * sum over p in a group with src(p) = s of dc[p] . b[g(p)]^T`.  The returned buffer is the call's
    /// scratch: keep it until the stream has passed the call.
    pub fn gemm_grad_a<T: RowScalar>(&self, flags: i32, alpha: f64, dc: &HipView<T>, b: &HipView<T>, da: &mut HipViewMut<T>, stream: &Stream) -> Result<HipBuffer<u8>> {
        let k = b.dims().get(1).copied().ok_or_else(|| Error::RankMismatch { expected: 3, got: b.dims().len() })?;
        let need = unsafe { sys::tfh_ragged_gemm_grad_a_workspace(T::TAG, self.n_rows as i64, k as i64, self.fan as i32, flags) };
        let scratch = HipBuffer::<u8>::new(need.max(1), self.offsets.device_id())?;
        let (g, dc, b, da) = (self.raw(), dc.raw(), b.raw(), da.raw());
        check(unsafe {
            sys::tfh_ragged_gemm_grad_a(
                T::TAG, &g, flags, alpha, &dc, &b, &da, scratch.as_device_ptr() as *mut c_void, need, stream.raw(),
            )
        })?;
        Ok(scratch)
    }

    /// `y[t] = sum_j weights[t, j] * x[positions[t * fan + j]]`.
    pub fn combine<T: RowScalar>(&self, x: &HipView<T>, weights: Option<&HipView<T::Sum>>, y: &mut HipViewMut<T>, stream: &Stream) -> Result<()> {
        let (g, x, w, y) = (self.raw(), x.raw(), optional(weights), y.raw());
        check(unsafe { sys::tfh_combine_rows(T::TAG, &g, &x, address(&w), &y, stream.raw()) })
    }

    /// The gradients of `combine`.
    pub fn combine_grad<T: RowScalar>(
        &self,
        x: &HipView<T>,
        weights: Option<&HipView<T::Sum>>,
        dy: &HipView<T>,
        dx: Option<&mut HipViewMut<T>>,
        dweights: Option<&mut HipViewMut<T::Sum>>,
        stream: &Stream,
    ) -> Result<()> {
        let (g, x, w, dy, dx, dw) = (self.raw(), x.raw(), optional(weights), dy.raw(), optional_mut(dx), optional_mut(dweights));
        check(unsafe {
            sys::tfh_combine_rows_grad(T::TAG, &g, &x, address(&w), &dy, address(&dx), address(&dw), stream.raw())
        })
    }

    fn workspace<T: RowScalar>(&self, rank: usize, gradient: bool) -> Result<(HipBuffer<u8>, usize)> {
        let need = unsafe { sys::tfh_adapter_workspace(T::TAG, self.n_rows as i64, rank as i64, gradient as i32) };
        Ok((HipBuffer::new(need.max(1), self.offsets.device_id())?, need))
    }

    fn rank_of<T: RowScalar>(factors: &AdapterFactors<T>) -> Result<usize> {
        factors.a.dims().get(2).copied().ok_or_else(|| Error::RankMismatch { expected: 3, got: factors.a.dims().len() })
    }

    /// `y[t] = x[t] . w + scales[g] * (x[t] . a[g]) . b[g]`.  The returned buffer is the call's scratch: keep it until
    /// the stream has passed the call.
    pub fn adapter_gemm<T: RowScalar>(&self, x: &HipView<T>, w: &HipView<T>, factors: &AdapterFactors<T>, y: &mut HipViewMut<T>, stream: &Stream) -> Result<HipBuffer<u8>> {
        let (scratch, need) = self.workspace::<T>(Self::rank_of(factors)?, false)?;
        let (g, x, w, a, b, s, y) = (self.raw(), x.raw(), w.raw(), factors.a.raw(), factors.b.raw(), optional(factors.scales), y.raw());
        check(unsafe {
            sys::tfh_adapter_gemm(
                T::TAG, &g, &x, &w, &a, &b, address(&s), &y, scratch.as_device_ptr() as *mut c_void, need, stream.raw(),
            )
        })?;
        Ok(scratch)
    }

    /// The gradients of `adapter_gemm` for a `w` that stays as it is; scratch as there.
    #[allow(clippy::too_many_arguments)]
    pub fn adapter_gemm_grad<T: RowScalar>(
        &self,
        x: &HipView<T>,
        w: &HipView<T>,
        factors: &AdapterFactors<T>,
        dy: &HipView<T>,
        dx: Option<&mut HipViewMut<T>>,
        da: Option<&mut HipViewMut<T>>,
        db: Option<&mut HipViewMut<T>>,
        stream: &Stream,
    ) -> Result<HipBuffer<u8>> {
        let (scratch, need) = self.workspace::<T>(Self::rank_of(factors)?, true)?;
        let (g, x, w, a, b, s) = (self.raw(), x.raw(), w.raw(), factors.a.raw(), factors.b.raw(), optional(factors.scales));
        let (dy, dx, da, db) = (dy.raw(), optional_mut(dx), optional_mut(da), optional_mut(db));
        check(unsafe {
            sys::tfh_adapter_gemm_grad(
                T::TAG, &g, &x, &w, &a, &b, address(&s), &dy, address(&dx), address(&da), address(&db),
                scratch.as_device_ptr() as *mut c_void, need, stream.raw(),
            )
        })?;
        Ok(scratch)
    }
}
